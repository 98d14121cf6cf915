// Scoring rows of logits in one pass: log probability of a given token, its rank, the row's entropy, and the best alternatives.
//
//   m = max x, S = sum exp(x - m), H = ln S - sum exp(x - m) (x - m) / S,  log p(t) = (x_t - m) - ln S
//   rank(t) = 1 + the tokens with a larger logit, or the same and a lower index
//
// A row is cut into parts, one wave each; a wave reads its part once, in batches of kBatch neighbouring logits, and keeps per lane the running maximum
// and the two sums, and across its lanes the sorted list of the best (lane i: the i-th).  Parts of a row are joined by a second launch.
//
// A logit is looked at for the list only where a batch holds one above the list's last; candidates enter in the order of their index,
// so a strict comparison leaves ties with the lower index.  Where a batch holds many (the first one; ascending logits), a bisection over the
// lanes' maxima first finds a value that at least n of the batch reach.
//
// -inf is a masked token: probability 0, no alternative.  A row of nothing else has log probability -inf, entropy 0 and no alternatives.  NaN or +inf in a
// row leaves NaN in log probability and entropy, as the formula does.  A row at the type's lowest value is an ordinary, uniform row.
#include "typed_rows.hpp"

#include <algorithm>

#pragma clang fp contract(off)

namespace cml {

constexpr float kLowest = -3.4028235e38f;
constexpr float kLog2e = 1.44269504088896341f, kLn2 = 0.693147180559945309f;
constexpr int kBatch = 1024;      // logits a wave takes at once: 16 a lane
constexpr int kMaxParts = 128;    // per row

struct ScoreArgs {
    const void *logits;
    const int32_t *target;
    float *log_prob, *entropy, *top_log_probs;
    int32_t *rank, *top_ids;
    float *partial;
    int64_t stride, n_rows;
    int vocab, n_top, parts;
};

__host__ __device__ constexpr int partial_floats(int n_top) { return 4 + 2 * n_top; }

// What a wave has seen of a row.  Per lane: most, sum, esum; the same in all lanes: above.
struct RowState {
    float most = kLowest;   // running maximum, never below the lowest finite value
    float sum = 0.0f;       // of exp(x - most)
    float esum = 0.0f;      // of exp(x - most) (x - most) log2(e)
    int above = 0;          // tokens ahead of the given one
    float list = -INFINITY; // lane i: the i-th best
    int list_id = -1;
};

// d as a factor: the exponential of one so low is 0, and 0 times a finite number adds nothing (a masked token, an overflowed difference).
__device__ __forceinline__ float finite_factor(float d) { return fmaxf(d, -1e25f); }

__device__ __forceinline__ void list_insert(RowState &s, float v, int id, int lane) {
    const int at = __builtin_popcountll(__builtin_amdgcn_ballot_w64(s.list >= v));
    const float up = dpp_f32<0x138>(s.list);  // wave_shr:1
    const int up_id = __builtin_amdgcn_update_dpp(0, s.list_id, 0x138, 0xf, 0xf, false);
    s.list = lane < at ? s.list : lane == at ? v : up;
    s.list_id = lane < at ? s.list_id : lane == at ? id : up_id;
}

// The running sums of a lane moved to another maximum.
__device__ __forceinline__ void rebase(RowState &s, float most) {
    const float d = (s.most - most) * kLog2e, f = __builtin_amdgcn_exp2f(d);
    s.esum = f * fmaf(s.sum, finite_factor(d), s.esum);
    s.sum = f * s.sum;  // (a NaN stays)
    s.most = most;
}

// A value that at least n of the 64 lanes' v reach, close to the n-th largest: bisection over the upper half of the ordered bits.
__device__ __forceinline__ float nth_bound(float v, int n) {
    const int key = total_key(v) >> 16;
    int low = -32768;
    for (int bit = 32768; bit; bit >>= 1)
        if (__builtin_popcountll(__builtin_amdgcn_ballot_w64(key >= low + bit)) >= n) low += bit;
    return from_total_key(static_cast<int>(static_cast<unsigned>(low) << 16));
}

// Sums over the lanes, every lane at the row's maximum.
__device__ __forceinline__ void close(RowState &s) {
    rebase(s, from_total_key(wave_allmax_i32(total_key(s.most))));
    s.sum = wave_allsum(s.sum);
    s.esum = wave_allsum(s.esum);
}

template <class T>
__device__ __forceinline__ void write_row(const ScoreArgs &a, int64_t row, const RowState &s, float given, bool in_range, int lane) {
    const float log_sum = __builtin_amdgcn_logf(s.sum) * kLn2;
    const bool empty = s.sum == 0.0f;
    if (lane == 0) {
        a.log_prob[row] = !in_range ? __builtin_nanf("") : empty ? -INFINITY : (given - s.most) - log_sum;
        if (a.rank) a.rank[row] = in_range ? s.above + 1 : 0;
        if (a.entropy) a.entropy[row] = empty ? 0.0f : log_sum - s.esum / s.sum * kLn2;
    }
    if (lane < a.n_top) {
        a.top_ids[row * a.n_top + lane] = s.list_id;
        a.top_log_probs[row * a.n_top + lane] = s.list_id < 0 ? -INFINITY : (s.list - s.most) - log_sum;
    }
}

template <class T>
__global__ __launch_bounds__(256) void token_log_probs_kernel(ScoreArgs a) {
    typedef typename T::Bits Bits;
    constexpr int EP = 8, U = kBatch / 64 / EP;  // a piece of eight logits a lane
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t id = static_cast<int64_t>(blockIdx.x) * 4 + wave;
    const int64_t row = id / a.parts;
    const int part = static_cast<int>(id - row * a.parts);
    if (row >= a.n_rows) return;
    const Bits *x = static_cast<const Bits *>(a.logits) + row * a.stride;
    const int target = a.target[row];
    const bool in_range = target >= 0 && target < a.vocab;
    const float given = in_range ? load_value<T>(x + target) : INFINITY;
    const int n_batches = (a.vocab + kBatch - 1) / kBatch;
    const int begin = static_cast<int>(static_cast<int64_t>(n_batches) * part / a.parts), end = static_cast<int>(static_cast<int64_t>(n_batches) * (part + 1) / a.parts);
    RowState s;
    float last = -INFINITY;  // the list's n-th
    for (int b = begin; b < end; b++) {
        const int base = b * kBatch;
        float v[U][EP];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int i = base + (u * 64 + lane) * EP;
            if (i + EP <= a.vocab) {
                load8<T>(x + i, v[u]);
            } else {
#pragma unroll
                for (int j = 0; j < EP; j++) v[u][j] = i + j < a.vocab ? load_value<T>(x + i + j) : -INFINITY;
            }
        }
        float bm = -INFINITY;
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int j = 0; j < EP; j++) bm = fmaxf(bm, v[u][j]);
        rebase(s, fmaxf(s.most, bm));
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int j = 0; j < EP; j++) {
                const float d = (v[u][j] - s.most) * kLog2e, e = __builtin_amdgcn_exp2f(d);
                s.sum = s.sum + e;
                s.esum = fmaf(e, finite_factor(d), s.esum);
                const int i = base + (u * 64 + lane) * EP + j;
                s.above += __builtin_popcountll(__builtin_amdgcn_ballot_w64(i < a.vocab && (v[u][j] > given || (v[u][j] == given && i < target))));
            }
        if (a.n_top == 0) continue;
        unsigned long long lanes = __builtin_amdgcn_ballot_w64(bm > last);
        if (!lanes) continue;
        float bound = -INFINITY;
        if (__builtin_popcountll(lanes) > a.n_top) bound = nth_bound(bm, a.n_top);
#pragma unroll
        for (int u = 0; u < U; u++) {
            float pm = v[u][0];
#pragma unroll
            for (int j = 1; j < EP; j++) pm = fmaxf(pm, v[u][j]);
            lanes = __builtin_amdgcn_ballot_w64(pm > last && pm >= bound);
            while (lanes) {
                const int from = __builtin_ctzll(lanes);
                lanes &= lanes - 1;
#pragma unroll
                for (int j = 0; j < EP; j++) {
                    const float c = lane_of(v[u][j], from);
                    if (c > last && c >= bound) {
                        list_insert(s, c, base + (u * 64 + from) * EP + j, lane);
                        last = lane_of(s.list, a.n_top - 1);
                    }
                }
            }
        }
    }
    close(s);
    if (a.parts == 1) {
        write_row<T>(a, row, s, given, in_range, lane);
    } else {
        float *p = a.partial + id * partial_floats(a.n_top);
        if (lane == 0) {
            p[0] = s.most;
            p[1] = s.sum;
            p[2] = s.esum;
            p[3] = __builtin_bit_cast(float, s.above);
        }
        if (lane < a.n_top) {
            p[4 + lane] = s.list;
            p[4 + a.n_top + lane] = __builtin_bit_cast(float, s.list_id);
        }
    }
}

// The parts of a row, joined by one wave: lane p takes the sums of parts p, p + 64, ...; the lists go in order.
template <class T>
__global__ __launch_bounds__(64) void token_log_probs_join_kernel(ScoreArgs a) {
    typedef typename T::Bits Bits;
    const int lane = threadIdx.x;
    const int64_t row = blockIdx.x;
    const int width = partial_floats(a.n_top);
    const float *p = a.partial + row * a.parts * width;
    RowState s;
    for (int i = lane; i < a.parts; i += 64) {
        RowState o;
        o.most = p[i * width];
        o.sum = p[i * width + 1];
        o.esum = p[i * width + 2];
        const float most = fmaxf(s.most, o.most);
        rebase(s, most);
        rebase(o, most);
        s.sum = s.sum + o.sum;
        s.esum = s.esum + o.esum;
        s.above += __builtin_bit_cast(int, p[i * width + 3]);
    }
    close(s);
    for (int o = 1; o < 64; o <<= 1) s.above += __shfl_xor(s.above, o);
    float last = -INFINITY;
    const int n = a.parts * a.n_top;
    for (int i0 = 0; i0 < n; i0 += 64) {
        const int i = min(i0 + lane, n - 1), part = i / a.n_top, at = i - part * a.n_top;
        const float v = i0 + lane < n ? p[part * width + 4 + at] : -INFINITY;
        const int id = __builtin_bit_cast(int, p[part * width + 4 + a.n_top + at]);
        unsigned long long lanes = __builtin_amdgcn_ballot_w64(v > last);
        while (lanes) {
            const int from = __builtin_ctzll(lanes);
            lanes &= lanes - 1;
            const float c = lane_of(v, from);
            if (c > last) {
                list_insert(s, c, __builtin_amdgcn_readlane(id, from), lane);
                last = lane_of(s.list, a.n_top - 1);
            }
        }
    }
    const int target = a.target[row];
    const bool in_range = target >= 0 && target < a.vocab;
    const float given = in_range ? load_value<T>(static_cast<const Bits *>(a.logits) + row * a.stride + target) : 0.0f;
    write_row<T>(a, row, s, given, in_range, lane);
}

// Parts per row: enough waves for the chip, one batch a part at least.
static int score_parts(int64_t n_rows, int64_t vocab) {
    const int64_t batches = (vocab + kBatch - 1) / kBatch;
    return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({(4096 + n_rows - 1) / n_rows, batches, kMaxParts})));
}

size_t token_log_probs_workspace(int64_t n_rows, int64_t vocab, int n_top) {
    const int parts = score_parts(n_rows, vocab);
    return parts == 1 ? 0 : static_cast<size_t>(n_rows) * parts * partial_floats(n_top) * sizeof(float);
}

int launch_token_log_probs(int dtype, const void *logits, int64_t stride, int64_t n_rows, int64_t vocab, const int32_t *target, int n_top, float *log_prob, int32_t *rank, float *entropy,
                           int32_t *top_ids, float *top_log_probs, void *workspace, hipStream_t st) {
    const ScoreArgs a{logits, target, log_prob, entropy, top_log_probs, rank, top_ids, static_cast<float *>(workspace), stride, n_rows, static_cast<int>(vocab), n_top, score_parts(n_rows, vocab)};
    return with_type(dtype, [&](auto t) {
        typedef decltype(t) T;
        CML_COUNT_LAUNCH("score.rows");
        hipLaunchKernelGGL(token_log_probs_kernel<T>, dim3(static_cast<unsigned>((n_rows * a.parts + 3) / 4)), dim3(256), 0, st, a);
        if (a.parts > 1) {
            CML_COUNT_LAUNCH("score.join");
            hipLaunchKernelGGL(token_log_probs_join_kernel<T>, dim3(static_cast<unsigned>(n_rows)), dim3(64), 0, st, a);
        }
        CML_HIP_TRY(hipGetLastError());
        return CML_OK;
    });
}

}  // namespace cml
