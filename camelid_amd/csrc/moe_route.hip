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
// A token has a whole wave, or 16 lanes of one.  A group has 1, 2, 4, 8 or 16 lanes and each of them NE neighbouring experts (the group's last ones fewer or none):
// what is ahead in lane and place has the lower index.  With 16 lanes for a token each has the experts of four, and adds them up as four, so that both forms give the
// same bits.
#include <algorithm>
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
    int group_shift;  // log2 of the lanes that hold a group
    int renormalise;
    float weight_scale;
};

constexpr int kOut = INT32_MIN;  // key of an expert that takes no part: below every ordered float

// The experts of a lane.
template <int NE>
struct LaneExperts {
    int first, count;
    __device__ __forceinline__ LaneExperts(const RouteArgs &a, int lane) {
        const int group = lane >> a.group_shift, at = (lane & ((1 << a.group_shift) - 1)) * NE;
        first = group * a.group_size + at;
        count = group < a.n_groups ? max(0, min(NE, a.group_size - at)) : 0;
    }
};

// Their values, -inf behind the last.
template <class T, int NE>
__device__ __forceinline__ void load_experts(const typename T::Bits *p, const LaneExperts<NE> &my, float (&v)[NE]) {
    if constexpr (NE >= 8) {
        if (my.count == NE) {
#pragma unroll
            for (int j = 0; j < NE; j += 8) {
                float eight[8];
                load8<T>(p + my.first + j, eight);
#pragma unroll
                for (int i = 0; i < 8; i++) v[j + i] = eight[i];
            }
            return;
        }
    }
#pragma unroll
    for (int j = 0; j < NE; j++) v[j] = -INFINITY;
    if (my.count > 0)
#pragma unroll
        for (int j = 0; j < NE; j++) {
            const float here = load_value<T>(p + my.first + min(j, my.count - 1));
            v[j] = j < my.count ? here : -INFINITY;
        }
}

// Scores and values (the floats behind the keys) of a lane's experts; LANES lanes have the token.  in: takes part; the value of one that does not is -inf.
template <class T, bool SIGMOID, int NE, int LANES>
__device__ __forceinline__ void rate_experts(const RouteArgs &a, int64_t t, const LaneExperts<NE> &my, float (&score)[NE], float (&value)[NE], bool (&in)[NE]) {
    float most = -3.4028235e38f;
    load_experts<T, NE>(static_cast<const typename T::Bits *>(a.logits) + t * a.stride, my, value);
#pragma unroll
    for (int j = 0; j < NE; j++) {
        in[j] = value[j] > -INFINITY;  // (false for NaN)
        value[j] = fminf(value[j], 3.4028235e38f);
        if (in[j]) most = fmaxf(most, value[j]);
    }
    if constexpr (SIGMOID) {
#pragma unroll
        for (int j = 0; j < NE; j++) score[j] = in[j] ? 1.0f / (1.0f + expf(-value[j])) : 0.0f;
    } else {
        most = from_total_key(LANES == 64 ? wave_allmax_i32(total_key(most)) : row_allmax_i32(total_key(most)));
        constexpr int kParts = 64 / LANES;
        float sum[kParts] = {};
#pragma unroll
        for (int j = 0; j < NE; j++) {
            score[j] = in[j] ? expf(value[j] - most) : 0.0f;
            sum[j / (NE / kParts)] = sum[j / (NE / kParts)] + score[j];
        }
        float total;
        if constexpr (LANES == 64) total = rows_allsum(sum[0]);
        else total = row_allsum((sum[0] + sum[1]) + (sum[2] + sum[3]));
        if (total > 0.0f)
#pragma unroll
            for (int j = 0; j < NE; j++) score[j] = score[j] / total;
    }
    if (a.bias) {
        float bias[NE];
        load_experts<TypeF32, NE>(a.bias, my, bias);
#pragma unroll
        for (int j = 0; j < NE; j++) value[j] = score[j] + bias[j];
    }
#pragma unroll
    for (int j = 0; j < NE; j++) {
        in[j] = in[j] && value[j] > -INFINITY;
        value[j] = in[j] ? value[j] + 0.0f : -INFINITY;  // (-0 is 0)
    }
}

// What a group is rated by: its best keys; without a bias and for two, the scores, which order as the logits do.
template <int NE>
__device__ __forceinline__ void group_keys(const RouteArgs &a, const float (&score)[NE], const float (&value)[NE], const bool (&in)[NE], int (&rated)[NE]) {
#pragma unroll
    for (int j = 0; j < NE; j++) rated[j] = in[j] ? total_key(a.bias || a.group_top == 1 ? value[j] : score[j]) : kOut;
}
__device__ __forceinline__ int group_worth(const RouteArgs &a, int first, int second) {
    if (first == kOut) return kOut;
    if (a.group_top == 1 || second == kOut) return first;
    return total_key(from_total_key(first) + from_total_key(second) + 0.0f);
}
// The worth of the group that a lane belongs to: two best per lane, then of pairs of lanes, of fours, ...
template <int NE>
__device__ __forceinline__ int lanes_worth(const RouteArgs &a, const int (&rated)[NE]) {
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
    if (a.group_shift >= 1) meet(std::integral_constant<int, 0xB1>{});   // quad_perm [1,0,3,2]
    if (a.group_shift >= 2) meet(std::integral_constant<int, 0x4E>{});   // quad_perm [2,3,0,1]
    if (a.group_shift >= 3) meet(std::integral_constant<int, 0x141>{});  // row_half_mirror: the other quad
    if (a.group_shift >= 4) meet(std::integral_constant<int, 0x140>{}); // row_mirror: the other eight
    return group_worth(a, first, second);
}

// A wave per token.  The logits are little to read; what it takes is instructions: a sigmoid's exponential and division are 25 for every expert, a turn of the
// choice about 30, so that 8 of 256 for 8192 tokens (4 MB) come to 11.6 us, where reading them takes 1.  One token: 8 of 128 3.2 us, most of it the launch, 8 of 256 in 8 groups 4.3.
template <class T, bool SIGMOID, int NE>
__global__ __launch_bounds__(256) void moe_route_scored_kernel(RouteArgs a) {
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int64_t t = static_cast<int64_t>(blockIdx.x) * 4 + wave;
    if (t >= a.n_tokens) return;  // (a wave's work is its own: no barriers)
    float score[NE], value[NE];
    bool in[NE];
    const LaneExperts<NE> my(a, lane);
    rate_experts<T, SIGMOID, NE, 64>(a, t, my, score, value, in);
    int key[NE];
#pragma unroll
    for (int j = 0; j < NE; j++) key[j] = in[j] ? total_key(value[j]) : kOut;
    if (a.n_groups > 1) {
        int rated[NE];
        group_keys(a, score, value, in, rated);
        const int worth = lanes_worth(a, rated), mine = lane >> a.group_shift;
        int ahead = 0;  // a group stays if fewer than groups_kept are ahead of it
        for (int g = 0; g < a.n_groups; g++) {
            const int theirs = __builtin_amdgcn_readlane(worth, g << a.group_shift);
            ahead += (theirs > worth) | ((theirs == worth) & (g < mine));
        }
        if (ahead >= a.groups_kept)
#pragma unroll
            for (int j = 0; j < NE; j++) key[j] = kOut;
    }
    int place = -1;  // lane s: where slot s is, its lane * NE + j
    for (int s = 0; s < a.k; s++) {
        int best = key[NE - 1], at = NE - 1;
#pragma unroll
        for (int j = NE - 2; j >= 0; j--) {
            at = key[j] >= best ? j : at;
            best = max(best, key[j]);
        }
        const int m = wave_allmax_i32(best);
        if (m == kOut) break;
        const int p = __builtin_amdgcn_readlane(lane * NE + at, __builtin_ctzll(__builtin_amdgcn_ballot_w64(best == m)));
#pragma unroll
        for (int j = 0; j < NE; j++) key[j] = p == lane * NE + j ? kOut : key[j];
        place = lane == s ? p : place;
    }
    // the chosen experts and their scores, from the lanes that hold them
    const int holder = (place < 0 ? 0 : place) / NE;
    const int chosen = place < 0 ? -1 : LaneExperts<NE>(a, holder).first + place % NE;
    float w = 0.0f;
#pragma unroll
    for (int j = 0; j < NE; j++) {
        const float theirs = __shfl(score[j], holder);
        w = place >= 0 && place % NE == j ? theirs : w;
    }
    if (a.renormalise) {
        const float sum = rows_allsum(w);
        const int live = __builtin_popcountll(__builtin_amdgcn_ballot_w64(chosen >= 0));
        w = sum > 0.0f ? w / sum : chosen >= 0 ? 1.0f / static_cast<float>(live) : 0.0f;  // (all chosen scores 0: alike)
    }
    if (lane < a.k) {
        a.idx[t * a.k + lane] = chosen;
        a.weight[t * a.k + lane] = w * a.weight_scale;
    }
}

// Four tokens a wave, 16 lanes each, for up to MOST of 16 * NE experts.  Every lane sorts its experts first, as doubles: a value's f32 bits are the upper word (finite
// and infinite floats are finite doubles, in the same order), its place the lower one, so that a comparison that the chip makes at full rate decides ties as well.
// Then the lanes' first entries meet k times, and the lane that held the best goes on to its next.  A turn's
// maximum over 16 lanes serves four tokens, so a token takes 340 instructions in place of some 600: 8 of 256 for 8192 tokens 8.1 us, two waves to a SIMD and bound by the
// latency of their chains; 16 of 512 15.0 us, 680 instructions, which issue in two thirds of the busy cycles.
__device__ __forceinline__ void sort_two(double &a, double &b) {  // descending
    const double hi = __builtin_fmax(a, b);
    b = __builtin_fmin(a, b);
    a = hi;
}
template <int N>
__device__ __forceinline__ void sort_bitonic(double *v) {
#pragma unroll
    for (int d = N / 2; d; d >>= 1)
#pragma unroll
        for (int i = 0; i < N; i++)
            if (!(i & d)) sort_two(v[i], v[i + d]);
}
// The first KEEP of N in order; what is behind them is left in any.
template <int N, int KEEP>
__device__ __forceinline__ void sort_best(double *v) {
    if constexpr (N == 4) {
        constexpr int kAt[5][2] = {{0, 1}, {2, 3}, {0, 2}, {1, 3}, {1, 2}};
#pragma unroll
        for (int i = 0; i < 5; i++) sort_two(v[kAt[i][0]], v[kAt[i][1]]);
    } else if constexpr (N == 8) {  // odd-even merges
        constexpr int kAt[19][2] = {{0, 1}, {2, 3}, {4, 5}, {6, 7}, {0, 2}, {1, 3}, {4, 6}, {5, 7}, {1, 2}, {5, 6}, {0, 4}, {1, 5}, {2, 6}, {3, 7}, {2, 4}, {3, 5}, {1, 2}, {3, 4}, {5, 6}};
#pragma unroll
        for (int i = 0; i < 19; i++) sort_two(v[kAt[i][0]], v[kAt[i][1]]);
    } else {
        sort_best<N / 2, KEEP>(v);
        sort_best<N / 2, KEEP>(v + N / 2);
        constexpr int kHalf = N / 2 < KEEP ? N / 2 : KEEP;  // sorted entries of a half
#pragma unroll
        for (int i = 0; i < kHalf; i++) sort_two(v[i], v[N / 2 + kHalf - 1 - i]);
        if constexpr (kHalf < KEEP) {  // both halves stay: what is behind the larger ones is theirs upside down
            sort_bitonic<kHalf>(v);
            sort_bitonic<kHalf>(v + kHalf);
        } else {
            sort_bitonic<kHalf>(v);
        }
    }
}

template <class T, bool SIGMOID, int NE, int MOST>
__global__ __launch_bounds__(256) void moe_route_scored_quarter_kernel(RouteArgs a) {
    constexpr int kEntries = NE < MOST ? NE : MOST;
    const int token = threadIdx.x >> 4, lane = threadIdx.x & 15;
    const int64_t t = static_cast<int64_t>(blockIdx.x) * 16 + token, here = min(t, a.n_tokens - 1);
    float score[NE], value[NE];
    bool in[NE];
    const LaneExperts<NE> my(a, lane);
    rate_experts<T, SIGMOID, NE, 16>(a, here, my, score, value, in);
    __shared__ __align__(16) float scores[16][16 * NE];  // (written and read by the same wave)
#pragma unroll
    for (int j = 0; j < NE; j++) scores[token][lane * NE + j] = score[j];
    if (a.n_groups > 1) {
        int rated[NE];
        group_keys(a, score, value, in, rated);
        const int worth = lanes_worth(a, rated), mine = lane >> a.group_shift;
        int ahead = 0;  // a group stays if fewer than groups_kept are ahead of it
        for (int g = 0; g < a.n_groups; g++) {
            const int theirs = __shfl(worth, g << a.group_shift, 16);
            ahead += (theirs > worth) | ((theirs == worth) & (g < mine));
        }
        if (ahead >= a.groups_kept)
#pragma unroll
            for (int j = 0; j < NE; j++) value[j] = -INFINITY;
    }
    double entry[NE];
#pragma unroll
    for (int j = 0; j < NE; j++) {
        const int bits = __builtin_bit_cast(int, value[j]);
        entry[j] = __hiloint2double(bits, ~((lane * NE + j) ^ (bits >> 31)));  // (of equal values the one ahead is the larger, of equal negative ones too)
    }
    sort_best<NE, kEntries>(entry);
    int key[kEntries], place[kEntries];
#pragma unroll
    for (int i = 0; i < kEntries; i++) {
        const int bits = __double2hiint(entry[i]);
        key[i] = total_key(__builtin_bit_cast(float, bits));
        place[i] = ~__double2loint(entry[i]) ^ (bits >> 31);
    }
    const int none = total_key(-INFINITY);
    int where = -1;  // lane s: slot s
#pragma unroll
    for (int s = 0; s < MOST; s++) {
        if (s == a.k) break;
        const int m = row_allmax_i32(key[0]);
        const int p = row_allmin_i32(key[0] == m ? place[0] : INT32_MAX);
        where = lane == s && m != none ? p : where;
        const bool next = place[0] == p;
#pragma unroll
        for (int i = 0; i < kEntries - 1; i++)
            if (i < MOST - 1 - s) {  // (what no later turn gets to stays)
                key[i] = next ? key[i + 1] : key[i];
                place[i] = next ? place[i + 1] : place[i];
            }
        if (s + kEntries < MOST) {
            key[kEntries - 1] = next ? none : key[kEntries - 1];
            place[kEntries - 1] = next ? INT32_MAX : place[kEntries - 1];
        }
    }
    const int chosen = where < 0 ? -1 : LaneExperts<NE>(a, where / NE).first + where % NE;
    float w = where >= 0 ? scores[token][where] : 0.0f;
    if (a.renormalise) {
        const float sum = row_allsum(w);
        const int live = __builtin_popcount(static_cast<unsigned>(__builtin_amdgcn_ballot_w64(chosen >= 0) >> (threadIdx.x & 48)) & 0xffffu);
        w = sum > 0.0f ? w / sum : chosen >= 0 ? 1.0f / static_cast<float>(live) : 0.0f;  // (all chosen scores 0: alike)
    }
    if (t < a.n_tokens && lane < a.k) {
        a.idx[t * a.k + lane] = chosen;
        a.weight[t * a.k + lane] = w * a.weight_scale;
    }
}

template <class T, bool SIGMOID, int NE>
static int launch_route_wave(const RouteArgs &a, hipStream_t st) {
    CML_COUNT_LAUNCH("moe.route.scored");
    hipLaunchKernelGGL((moe_route_scored_kernel<T, SIGMOID, NE>), dim3(static_cast<unsigned>((a.n_tokens + 3) / 4)), dim3(256), 0, st, a);
    CML_HIP_TRY(hipGetLastError());
    return CML_OK;
}
template <class T, bool SIGMOID, int NE, int MOST>
static int launch_route_quarter(const RouteArgs &a, hipStream_t st) {
    CML_COUNT_LAUNCH("moe.route.scored.quarter");
    hipLaunchKernelGGL((moe_route_scored_quarter_kernel<T, SIGMOID, NE, MOST>), dim3(static_cast<unsigned>((a.n_tokens + 15) / 16)), dim3(256), 0, st, a);
    CML_HIP_TRY(hipGetLastError());
    return CML_OK;
}
template <class T, bool SIGMOID, int MOST>
static int launch_route_quarters(const RouteArgs &a, int ne, hipStream_t st) {
    if (ne == 4) return launch_route_quarter<T, SIGMOID, 4, MOST>(a, st);
    if (ne == 8) return launch_route_quarter<T, SIGMOID, 8, MOST>(a, st);
    if (ne == 16) return launch_route_quarter<T, SIGMOID, 16, MOST>(a, st);
    return launch_route_quarter<T, SIGMOID, 32, MOST>(a, st);
}
template <class T, bool SIGMOID>
static int launch_route(RouteArgs a, hipStream_t st) {
    // The groups over 64 lanes: a power of two each, 16 at most (what rates them stays inside 16 lanes), and a power of two of experts for every lane; 1024 experts
    // in up to 64 groups come to 32 at most.
    a.group_shift = 0;
    while (a.n_groups << (a.group_shift + 1) <= 64 && (a.group_shift < 4 || a.n_groups == 1)) a.group_shift++;
    int ne = 1;
    while (ne << a.group_shift < a.group_size) ne *= 2;
    // Four tokens a wave where there are waves enough that way (8 of 256 in 8 groups, four against one: 1024 tokens 6.6 and 5.3 us, 4096 6.7 and 7.5, 8192 8.1
    // and 11.6; 16 of 512, 8192 tokens: 15.0 and 21.0).
    if (a.n_tokens >= env_int("CAMELID_HIP_ROUTE_QUARTER", 4096) && a.k <= 16 && a.group_shift >= 2 && ne <= 8) {
        a.group_shift -= 2;
        return a.k <= 8 ? launch_route_quarters<T, SIGMOID, 8>(a, 4 * ne, st) : launch_route_quarters<T, SIGMOID, 16>(a, 4 * ne, st);
    }
    if (ne == 1) return launch_route_wave<T, SIGMOID, 1>(a, st);
    if (ne == 2) return launch_route_wave<T, SIGMOID, 2>(a, st);
    if (ne == 4) return launch_route_wave<T, SIGMOID, 4>(a, st);
    if (ne == 8) return launch_route_wave<T, SIGMOID, 8>(a, st);
    if (ne == 16) return launch_route_wave<T, SIGMOID, 16>(a, st);
    return launch_route_wave<T, SIGMOID, 32>(a, st);
}

int launch_moe_route_scored(int score, int dtype, const void *logits, int64_t stride, const float *bias, int64_t n_tokens, int n_experts, int n_groups, int groups_kept, int group_top, int k,
                            int renormalise, float weight_scale, int32_t *idx, float *weight, hipStream_t st) {
    const int size = n_experts / n_groups;
    const int64_t most = 4 * most_workgroups(256);  // tokens of a launch, a wave each
    return with_type(dtype, [&](auto t) {
        typedef decltype(t) T;
        for (int64_t first = 0; first < n_tokens; first += most) {
            const RouteArgs a{static_cast<const typename T::Bits *>(logits) + first * stride, bias, idx + first * k, weight + first * k, stride, std::min(most, n_tokens - first), n_experts, n_groups,
                              groups_kept, group_top, k, size, 0, renormalise, weight_scale};
            if (int rc = score == CML_ROUTE_SIGMOID ? launch_route<T, true>(a, st) : launch_route<T, false>(a, st)) return rc;
        }
        return CML_OK;
    });
}

}  // namespace cml
