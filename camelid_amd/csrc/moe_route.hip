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
        // groups one after the other, each lane's experts of that group against the wave
        unsigned long long kept = 0;
        int worth = kOut;  // of group `lane`
        for (int g = 0; g < a.n_groups; g++) {
            float sum = 0.0f;
            bool any = false;
            int taken = -1;
            for (int s = 0; s < a.group_top; s++) {
                int best = kOut;
#pragma unroll
                for (int j = 0; j < NE; j++) {
                    const int e = lane * NE + j;
                    if (static_cast<int>(e * a.size_inverse >> 20) == g && e != taken) best = max(best, key[j]);
                }
                const int m = wave_allmax_i32(best);
                if (m == kOut) break;
                int mine = -1;
                float sc = 0.0f;
#pragma unroll
                for (int j = NE - 1; j >= 0; j--) {
                    const int e = lane * NE + j;
                    if (static_cast<int>(e * a.size_inverse >> 20) == g && e != taken && key[j] == m) {
                        mine = e;
                        sc = score[j];
                    }
                }
                const int from = __builtin_ctzll(__builtin_amdgcn_ballot_w64(mine >= 0));
                taken = __builtin_amdgcn_readlane(mine, from);
                sum = sum + (a.bias || a.group_top == 1 ? from_total_key(m) : lane_of(sc, from));
                any = true;
            }
            if (lane == g && any) worth = total_key(sum + 0.0f);
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
    int chosen = -1;  // lane s: slot s
    float w = 0.0f;
    for (int s = 0; s < a.k; s++) {
        int best = kOut, at = 0;
        float sc = 0.0f;
#pragma unroll
        for (int j = NE - 1; j >= 0; j--)
            if (key[j] >= best) {
                best = key[j];
                at = j;
                sc = score[j];
            }
        const int m = wave_allmax_i32(best);
        if (m == kOut) break;
        const int from = __builtin_ctzll(__builtin_amdgcn_ballot_w64(best == m));
        const int e = __builtin_amdgcn_readlane(lane * NE + at, from);
        const float es = lane_of(sc, from);
#pragma unroll
        for (int j = 0; j < NE; j++)
            if (lane * NE + j == e) key[j] = kOut;
        if (lane == s) {
            chosen = e;
            w = es;
        }
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

template <class T, bool SIGMOID>
static int launch_route(const RouteArgs &a, hipStream_t st) {
    const dim3 grid(static_cast<unsigned>((a.n_tokens + 3) / 4)), block(256);
    if (a.n_experts <= 64) hipLaunchKernelGGL((moe_route_scored_kernel<T, SIGMOID, 1>), grid, block, 0, st, a);
    else if (a.n_experts <= 128) hipLaunchKernelGGL((moe_route_scored_kernel<T, SIGMOID, 2>), grid, block, 0, st, a);
    else if (a.n_experts <= 256) hipLaunchKernelGGL((moe_route_scored_kernel<T, SIGMOID, 4>), grid, block, 0, st, a);
    else if (a.n_experts <= 512) hipLaunchKernelGGL((moe_route_scored_kernel<T, SIGMOID, 8>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((moe_route_scored_kernel<T, SIGMOID, 16>), grid, block, 0, st, a);
    CML_HIP_TRY(hipGetLastError());
    return CML_OK;
}

int launch_moe_route_scored(int score, int dtype, const void *logits, int64_t stride, const float *bias, int64_t n_tokens, int n_experts, int n_groups, int groups_kept, int group_top, int k,
                            int renormalise, float weight_scale, int32_t *idx, float *weight, hipStream_t st) {
    const int size = n_experts / n_groups;
    const RouteArgs a{logits, bias, idx, weight, stride, n_tokens, n_experts, n_groups, groups_kept, group_top, k, size, ((1u << 20) + size - 1) / size, renormalise, weight_scale};
    CML_COUNT_LAUNCH("moe.route.scored");
    return with_type(dtype, [&](auto t) { return score == CML_ROUTE_SIGMOID ? launch_route<decltype(t), true>(a, st) : launch_route<decltype(t), false>(a, st); });
}

}  // namespace cml
