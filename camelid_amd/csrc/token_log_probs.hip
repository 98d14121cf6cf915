// Scoring rows of logits in one pass: log probability of a given token, its rank, the row's entropy, and the best alternatives.
//
//   m = max x, S = sum exp(x - m), H = ln S - sum exp(x - m) (x - m) / S,  log p(t) = (x_t - m) - ln S
//   rank(t) = 1 + the tokens with a larger logit, or the same and a lower index
//
// A row is cut into parts, one wave each; a wave reads its part once, in batches of neighbouring logits (the next one requested before this one is looked
// at), and keeps per lane the running maximum and the two sums, and across its lanes the sorted list of the best (lane i: the i-th).  Parts of a
// row are joined inside the workgroup where it has them all, else by a second launch.
//
// Logits are looked at one by one for the list only where a batch holds one above the list's last.  Where it holds many (the first one; ascending
// logits), a bisection over the lanes' maxima first finds a value that at least n of the batch reach, and one over all its logits where that leaves too many.
//
// Rows are to be read once, at memory's rate: 2048 x 128256 bf16 in 94 us without a list (5.6 TB/s), 114 with 20 best; what bounds the latter is instruction issue, 11
// to a logit and 80 insertions a part.  With fewer rows the lists weigh more, since every part fills one of its own: 512 rows 32 us without a list (4.1 TB/s), 35 with one best, 39 with 5, 50 with 20.  One row of 128256 f32 and 20 best: 11.0 us, two launches of which each waits for memory once.
//
// -inf is a masked token: probability 0, no alternative.  A row of nothing else has log probability -inf, entropy 0 and no alternatives.  NaN or +inf in a
// row leaves NaN in log probability and entropy, as the formula does.  A row at the type's lowest value is an ordinary, uniform row.
#include "typed_rows.hpp"

#include <algorithm>

#pragma clang fp contract(off)

namespace cml {

constexpr float kLowest = -3.4028235e38f;
constexpr float kLog2e = 1.44269504088896341f, kLn2 = 0.693147180559945309f;
constexpr int kMaxParts = 128;  // per row: two for a lane of the joining wave
constexpr int kJoinThreads = 512;

struct ScoreArgs {
    const void *logits;
    const int32_t *target;
    float *log_prob, *entropy, *top_log_probs;
    int32_t *rank, *top_ids;
    float *partial;
    int64_t stride, n_rows;
    int vocab, n_top, parts;
    int depth;             // which of the parts' entries bounds the row's n-th: with twice as many as n of them, half of the parts have n together
    uint32_t top_inverse;  // ceil(2^20 / n_top): i / n_top = i * top_inverse >> 20 for i < 8192
};

// most, sum, esum, above, the given logit; the list, value and id by turns
__host__ __device__ constexpr int partial_floats(int n_top) { return 5 + 2 * n_top; }

// What a wave has seen of a row.  Per lane: most, sum, esum; the same in all lanes: above.
struct RowState {
    float most = kLowest;   // running maximum, never below the lowest finite value
    float sum = 0.0f;       // of 2^d, d = (x - most) log2(e) + shift(most)
    float esum = 0.0f;      // of 2^d d
    int above = 0;          // tokens ahead of the given one
    uint32_t list = 0, list_low = 0;  // lane i: the i-th best, by the value's ordered bits, then the inverted id; 0: none
};

// What rounding most * log2(e) takes off it, for logits of ordinary size.  With it, d is one multiply-add, x log2(e) - rounded(most log2(e)), and as good as from the
// difference x - most; it goes out of the row's sums at their end.
constexpr float kOrdinary = 4096.0f;
__device__ __forceinline__ float shift(float most) { return fabsf(most) < kOrdinary ? fmaf(most, kLog2e, -(most * kLog2e)) : 0.0f; }

// d as a factor: the exponential of one so low is 0, and 0 times a finite number adds nothing (a masked token, an overflowed difference).
__device__ __forceinline__ float finite_factor(float d) { return fmaxf(d, -1e25f); }

// A finite or infinite f32 as an unsigned integer that orders like it (-0 as 0), above 0, and back.
__device__ __forceinline__ uint32_t ordered(uint32_t bits) {
    bits = bits == 0x80000000u ? 0u : bits;
    return bits ^ (static_cast<uint32_t>(static_cast<int>(bits) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float from_ordered(uint32_t v) { return v == 0 ? -INFINITY : __uint_as_float(v & 0x80000000u ? v ^ 0x80000000u : ~v); }

// Into its place by value, then by id; what falls off lane 63 is gone.  Every lane decides for itself, from its entry and the one before it.  (What an
// insertion takes is its instructions: 20 in front of every list of 20, 60 to 100 a part.)
__device__ __forceinline__ void list_insert(RowState &s, uint32_t v, int id) {
    const uint64_t c = static_cast<uint64_t>(v) << 32 | static_cast<uint32_t>(~id), mine = static_cast<uint64_t>(s.list) << 32 | s.list_low;
    const uint32_t up = __builtin_amdgcn_update_dpp(-1, s.list, 0x138, 0xf, 0xf, false), up_low = __builtin_amdgcn_update_dpp(-1, s.list_low, 0x138, 0xf, 0xf, false);  // wave_shr:1, all ones in lane 0
    const bool stays = mine > c, after = (static_cast<uint64_t>(up) << 32 | up_low) > c;
    s.list = stays ? s.list : after ? v : up;
    s.list_low = stays ? s.list_low : after ? static_cast<uint32_t>(~id) : up_low;
}
// The list from entries in any order, one a lane, `count` of them in the first lanes and 0 behind: each goes to the place that the number of larger ones says.
__device__ __forceinline__ void list_rank(RowState &s, uint2 mine, int count) {
    const uint64_t key = static_cast<uint64_t>(mine.x) << 32 | mine.y;
    int rank = 0;  // (a lane without an entry: the place behind the last)
    for (int i = 0; i < count; i++) {
        const uint64_t other = static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(mine.x, i))) << 32 | static_cast<uint32_t>(__builtin_amdgcn_readlane(mine.y, i));
        rank += other > key ? 1 : 0;
    }
    s.list = __builtin_amdgcn_ds_permute(4 * rank, mine.x);
    s.list_low = __builtin_amdgcn_ds_permute(4 * rank, mine.y);
}
// The running sums of a lane moved to another maximum.
__device__ __forceinline__ void rebase(RowState &s, float most) {
    const float d = (s.most - most) * kLog2e + (shift(most) - shift(s.most)), f = __builtin_amdgcn_exp2f(d);
    s.esum = f * fmaf(s.sum, finite_factor(d), s.esum);
    s.sum = f * s.sum;  // (a NaN stays)
    s.most = most;
}

// How many of the 64 K values v are above x.
template <int K>
__device__ __forceinline__ int count_above(const float (&v)[K], float x) {
    int above = 0;
#pragma unroll
    for (int k = 0; k < K; k++) above += __builtin_popcountll(__builtin_amdgcn_ballot_w64(v[k] > x));
    return above;
}
// A value that at least n of them are above, close below the n-th largest: bisection over the upper half of the ordered bits.  At least n have to be above -inf.
template <int K>
__device__ __forceinline__ float below_nth(const float (&v)[K], int n) {
    int low = -32768;
    const auto under = [](int half) __attribute__((always_inline)) {
        const int key = static_cast<int>(static_cast<unsigned>(half) << 16) - 1;
        return from_total_key(key == -1 ? -2 : key);  // (-0 is not below 0)
    };
    if constexpr (K <= 2) {
        int key[K];
#pragma unroll
        for (int k = 0; k < K; k++) key[k] = total_key(v[k]) >> 16;
        for (int bit = 32768; bit; bit >>= 1) {
            int reach = 0;
#pragma unroll
            for (int k = 0; k < K; k++) reach += __builtin_popcountll(__builtin_amdgcn_ballot_w64(key[k] >= low + bit));
            if (reach >= n) low += bit;
        }
    } else {
#pragma unroll 1
        for (int bit = 32768; bit; bit >>= 1)
            if (count_above(v, under(low + bit)) >= n) low += bit;  // (past the infinities: NaN, above which is nothing)
    }
    return under(low);
}

// Sums over the lanes, every lane at the row's maximum.
__device__ __forceinline__ void close(RowState &s) {
    rebase(s, from_total_key(wave_allmax_i32(total_key(s.most))));
    s.sum = wave_allsum(s.sum);
    s.esum = wave_allsum(s.esum);
}

// The largest logit's own term is 2^shift, the same instruction's result as in the sums, and goes out of them before anything is rounded: S is the sum divided by it, 1 or more, and
// what is left for the entropy is the other tokens'.  So no log probability is above 0 and no entropy below, and a row with one token left has 0 and 0.
template <class T>
__device__ __forceinline__ void write_row(const ScoreArgs &a, int64_t row, const RowState &s, float given, bool in_range, int lane) {
    const float more = shift(s.most), own = __builtin_amdgcn_exp2f(more);
    const float all = __builtin_amdgcn_logf(s.sum / own), log_sum = all * kLn2;
    const float entropy = (all - ((s.esum - own * more) - more * (s.sum - own)) / s.sum) * kLn2;
    const bool empty = s.sum == 0.0f;
    if (lane == 0) {
        a.log_prob[row] = !in_range ? __builtin_nanf("") : empty ? -INFINITY : (given - s.most) - log_sum;
        if (a.rank) a.rank[row] = in_range ? s.above + 1 : 0;
        if (a.entropy) a.entropy[row] = empty ? 0.0f : entropy;
    }
    if (lane < a.n_top) {
        a.top_ids[row * a.n_top + lane] = s.list ? static_cast<int>(~s.list_low) : -1;
        a.top_log_probs[row * a.n_top + lane] = s.list ? (from_ordered(s.list) - s.most) - log_sum : -INFINITY;
    }
}

// A lane's logits of a batch: pieces of eight, 64 lanes apart.
template <class T>
struct Batch {
    static constexpr int kPieces = sizeof(typename T::Bits) == 4 ? 2 : 4, kLogits = 64 * 8 * kPieces;
    v4u_row raw[kPieces * (sizeof(typename T::Bits) == 4 ? 2 : 1)];

    __device__ __forceinline__ void request(const typename T::Bits *p) {  // p: the lane's first logit
        typedef uint32_t v4u __attribute__((ext_vector_type(4), aligned(2)));
        constexpr int kPer = sizeof(typename T::Bits) == 4 ? 2 : 1;
#pragma unroll
        for (int u = 0; u < kPieces; u++)
#pragma unroll
            for (int k = 0; k < kPer; k++) raw[u * kPer + k] = __builtin_nontemporal_load(reinterpret_cast<const v4u *>(p + u * 512) + k);
    }
    __device__ __forceinline__ void take(float (&v)[kPieces][8]) const {
#pragma unroll
        for (int u = 0; u < kPieces; u++)
#pragma unroll
            for (int j = 0; j < 8; j++) {
                if constexpr (sizeof(typename T::Bits) == 4) v[u][j] = __uint_as_float(raw[2 * u + j / 4][j % 4]);
                else v[u][j] = T::widen(j & 1 ? raw[u][j / 2] >> 16 : raw[u][j / 2] & 0xffffu);
            }
    }
};

// INSIDE: 1, 2 or 4 parts a row, all of them in one workgroup.
template <class T, bool INSIDE>
__global__ __launch_bounds__(256) void token_log_probs_kernel(ScoreArgs a) {
    typedef typename T::Bits Bits;
    __shared__ uint2 found[INSIDE ? 1 : 4][64];
    constexpr int U = Batch<T>::kPieces, kBatch = Batch<T>::kLogits;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t id = blockIdx.x * 4 + wave, row = id / static_cast<uint32_t>(a.parts), part = id - row * a.parts;
    const bool live = row < a.n_rows;
    if (!live && !INSIDE) return;
    const Bits *x = static_cast<const Bits *>(a.logits) + (live ? row : 0) * a.stride;
    const int n_batches = (a.vocab + kBatch - 1) / kBatch;
    const int begin = static_cast<int>(static_cast<int64_t>(n_batches) * part / a.parts), end = live ? static_cast<int>(static_cast<int64_t>(n_batches) * (part + 1) / a.parts) : 0;
    Batch<T> ahead;
    const Bits *mine = x + lane * 8;
    // The row's last batch, where it is not whole: of a 16-bit type read from where a whole one ends with the row, what belongs to the batch before masked (one row of 128256 bf16,
    // 20 best: 13.5 us, logit by logit 15.5); of f32 logit by logit (half as many, and a request behind every batch, whole or not, costs more: 2048 x 128256 186 us and 223).
    constexpr bool kBack = sizeof(Bits) == 2;
    const bool fits = kBack && a.vocab >= kBatch;
    const int last_first = a.vocab - kBatch;
    if (begin < end) {
        if (fits) ahead.request(mine + min(begin * kBatch, last_first));
        else if ((begin + 1) * kBatch <= a.vocab) ahead.request(mine + begin * kBatch);
    }
    const int target = live ? a.target[row] : -1;
    const bool in_range = target >= 0 && target < a.vocab;
    const float given = in_range ? load_value<T>(x + target) : INFINITY;
    RowState s;
    float last = -INFINITY;  // the list's n-th
    bool careful = false;    // masked logits were seen
#pragma unroll 1
    for (int b = begin; b < end; b++) {
        const int base = b * kBatch;
        const bool whole = base + kBatch <= a.vocab;
        float v[U][8];
        // vmcnt(0): the batch is here.  Said outright, because the compiler, which does not see that no path leaves it in flight, otherwise waits below, at
        // reused registers, for the next batch as well (512 x 128256 bf16 63 us).
        __builtin_amdgcn_s_waitcnt(0x0f70);
        int first = base;
        if (fits) {
            ahead.take(v);
            if (b + 1 < end) ahead.request(mine + min(base + kBatch, last_first));
            if (!whole) {
                first = last_first;
#pragma unroll
                for (int u = 0; u < U; u++)
#pragma unroll
                    for (int j = 0; j < 8; j++) v[u][j] = first + (u * 64 + lane) * 8 + j >= base ? v[u][j] : -INFINITY;
            }
        } else if (!kBack && whole) {
            ahead.take(v);
            if (b + 1 < end && base + 2 * kBatch <= a.vocab) ahead.request(mine + base + kBatch);
        } else {
#pragma unroll
            for (int u = 0; u < U; u++)
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const int i = base + (u * 64 + lane) * 8 + j;
                    v[u][j] = i < a.vocab ? load_value<T>(x + i) : -INFINITY;
                }
        }
        float pm[U], bm = -INFINITY;
#pragma unroll
        for (int u = 0; u < U; u++) {
            pm[u] = fmaxf(fmaxf(fmaxf(v[u][0], v[u][1]), fmaxf(v[u][2], v[u][3])), fmaxf(fmaxf(v[u][4], v[u][5]), fmaxf(v[u][6], v[u][7])));
            bm = fmaxf(bm, pm[u]);
        }
        rebase(s, fmaxf(s.most, bm));
        // (instructions bound a row that comes at memory's rate: one less to a logit, and no clamp, is 2048 x 128256 bf16 in 113 us in place of 122)
        bool plain = whole && !careful && !__builtin_amdgcn_ballot_w64(!(fabsf(s.most) < kOrdinary));
        float sum = 0.0f, esum = 0.0f;  // (of this batch: a row's sum is one of few large terms)
        if (plain) {
            const float from = -(s.most * kLog2e);
#pragma unroll
            for (int u = 0; u < U; u++)
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const float d = fmaf(v[u][j], kLog2e, from), e = __builtin_amdgcn_exp2f(d);
                    sum = sum + e;
                    esum = fmaf(e, d, esum);
                }
            careful = __builtin_amdgcn_ballot_w64(esum != esum) != 0;  // a masked logit (0 times -inf), or a NaN: this batch again, and the rest of the part so
            plain = !careful;
        }
        if (!plain) {
            const float more = shift(s.most);
            sum = esum = 0.0f;
#pragma unroll
            for (int u = 0; u < U; u++)
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const float d = (v[u][j] - s.most) * kLog2e + more, e = __builtin_amdgcn_exp2f(d);
                    sum = sum + e;
                    esum = fmaf(e, finite_factor(d), esum);
                }
        }
        s.sum = s.sum + sum;
        s.esum = s.esum + esum;
        // tokens ahead of the given one: of equal logits those with a lower index (a given token is mostly among the first, and a batch without any ahead of it is
        // passed over)
        if (!__builtin_amdgcn_ballot_w64(bm >= given)) {
        } else if (whole && base + kBatch <= target) {
#pragma unroll
            for (int u = 0; u < U; u++)
#pragma unroll
                for (int j = 0; j < 8; j++) s.above += __builtin_popcountll(__builtin_amdgcn_ballot_w64(v[u][j] >= given));
        } else if (whole && base > target) {
#pragma unroll
            for (int u = 0; u < U; u++)
#pragma unroll
                for (int j = 0; j < 8; j++) s.above += __builtin_popcountll(__builtin_amdgcn_ballot_w64(v[u][j] > given));
        } else {
#pragma unroll
            for (int u = 0; u < U; u++)
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const int i = first + (u * 64 + lane) * 8 + j;
                    s.above += __builtin_popcountll(__builtin_amdgcn_ballot_w64(i >= base && i < a.vocab && (v[u][j] > given || (v[u][j] == given && i < target))));
                }
        }
        if (a.n_top == 0) continue;
        if (!__builtin_amdgcn_ballot_w64(bm > last)) continue;
        // (what the list holds has lower indices than this batch: only larger logits get in)
        const float most[1] = {bm};
        float over = last;
        if (__builtin_popcountll(__builtin_amdgcn_ballot_w64(bm > over)) > a.n_top + 8) over = fmaxf(over, below_nth(most, a.n_top));  // (the search takes what eight insertions do)
        const int lanes = __builtin_popcountll(__builtin_amdgcn_ballot_w64(bm > over));
        if (!whole || lanes >= 32) {  // lanes with many above it: a search among all of them takes what 80 insertions do
            const float (&all)[8 * U] = *reinterpret_cast<const float(*)[8 * U]>(&v);
            if (count_above(all, over) > (INSIDE ? a.n_top + 80 : 64)) over = fmaxf(over, below_nth(all, a.n_top));
        }
        if (!INSIDE && lanes > 12) {
            // Few rows, and the wave has the unit to itself: an insertion takes 60 ns, one after the other; gathered and ranked at once, 28 are 0.9 us instead of 1.7.
            int count = 0;
#pragma unroll
            for (int u = 0; u < U; u++) {
                if (!__builtin_amdgcn_ballot_w64(pm[u] > over)) continue;
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const bool in = v[u][j] > over;
                    const unsigned long long those = __builtin_amdgcn_ballot_w64(in);
                    const int at = count + __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(those >> 32), __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(those), 0));
                    if (in && at < 64) found[wave][at] = make_uint2(ordered(__float_as_uint(v[u][j])), static_cast<uint32_t>(~(first + (u * 64 + lane) * 8 + j)));
                    count += __builtin_popcountll(those);
                }
            }
            const int have = min(a.n_top, __builtin_popcountll(__builtin_amdgcn_ballot_w64(s.list != 0)));
            if (have + count <= 64) {
                __builtin_amdgcn_wave_barrier();
                const uint2 next = found[wave][max(lane - have, 0)];
                __builtin_amdgcn_wave_barrier();
                uint2 mine = make_uint2(0, 0);
                if (lane < have) mine = make_uint2(s.list, s.list_low);
                else if (lane < have + count) mine = next;
                list_rank(s, mine, have + count);
                last = from_ordered(__builtin_amdgcn_readlane(s.list, a.n_top - 1));
                continue;
            }
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (!__builtin_amdgcn_ballot_w64(pm[u] > over)) continue;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                unsigned long long in = __builtin_amdgcn_ballot_w64(v[u][j] > over);
                while (in) {
                    const int from = __builtin_ctzll(in);
                    in &= in - 1;
                    list_insert(s, ordered(__builtin_amdgcn_readlane(__float_as_uint(v[u][j]), from)), first + (u * 64 + from) * 8 + j);
                }
            }
        }
        last = from_ordered(__builtin_amdgcn_readlane(s.list, a.n_top - 1));
    }
    close(s);
    if constexpr (INSIDE) {
        __shared__ float sums[4][3];
        __shared__ int aboves[4];
        __shared__ uint2 lists[4][64];
        if (part > 0) {
            if (lane == 0) {
                sums[wave][0] = s.most;
                sums[wave][1] = s.sum;
                sums[wave][2] = s.esum;
                aboves[wave] = s.above;
            }
            lists[wave][lane] = make_uint2(s.list, s.list_low);
        }
        __syncthreads();
        if (part > 0 || !live) return;
        for (int p = wave + 1; p < wave + a.parts; p++) {
            RowState o;
            o.most = sums[p][0];
            o.sum = sums[p][1];
            o.esum = sums[p][2];
            const float most = fmaxf(s.most, o.most);
            rebase(s, most);
            rebase(o, most);
            s.sum = s.sum + o.sum;
            s.esum = s.esum + o.esum;
            s.above += aboves[p];
            if (a.n_top == 0) continue;
            const uint2 theirs = lists[p][lane];
            // (of equal logits those of this list have the lower ids)
            unsigned long long in = __builtin_amdgcn_ballot_w64(theirs.x > static_cast<uint32_t>(__builtin_amdgcn_readlane(s.list, a.n_top - 1)));
            while (in) {
                const int from = __builtin_ctzll(in);
                in &= in - 1;
                list_insert(s, __builtin_amdgcn_readlane(theirs.x, from), ~__builtin_amdgcn_readlane(theirs.y, from));
            }
        }
        write_row<T>(a, row, s, given, in_range, lane);
    } else {
        float *p = a.partial + static_cast<int64_t>(id) * partial_floats(a.n_top);
        if (lane == 0) {
            p[0] = s.most;
            p[1] = s.sum;
            p[2] = s.esum;
            p[3] = __builtin_bit_cast(float, s.above);
            p[4] = given;
        }
        if (lane < a.n_top) {
            p[5 + 2 * lane] = from_ordered(s.list);
            p[6 + 2 * lane] = __uint_as_float(~s.list_low);
        }
    }
}

// The parts of a row, joined: every thread asks for its share of the lists and every wave for the parts' best at once, so that memory is waited for once.  What
// reaches the n-th largest of the parts' best (of their `depth` best, where the parts are few) is gathered in LDS and ranked there (3 instructions for each, an insertion takes 20); the first wave adds the sums up
// (lane p: parts p and p + 64) and writes.  One row of 126 parts: 5 us with 20 best, 2.6 without a list, most of it the launch and the trip.
template <class T>
__global__ __launch_bounds__(kJoinThreads) void token_log_probs_join_kernel(ScoreArgs a) {
    __shared__ uint2 found[kJoinThreads], sorted[64];
    __shared__ int n_found;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int64_t row = blockIdx.x;
    const int width = partial_floats(a.n_top), n = a.parts * a.n_top;
    const float *rows = a.partial + row * a.parts * width;
    typedef uint32_t v2u __attribute__((ext_vector_type(2), aligned(4)));
    const auto entry = [&](int i) __attribute__((always_inline)) {
        const int part = static_cast<int>(static_cast<uint32_t>(i) * a.top_inverse >> 20);
        return *reinterpret_cast<const v2u *>(rows + part * width + 5 + 2 * (i - part * a.n_top));
    };
    constexpr int kMine = kMaxParts * 64 / kJoinThreads;
    v2u mine[kMine];
#pragma unroll
    for (int k = 0; k < kMine; k++)
        if (k * kJoinThreads < n) mine[k] = entry(min(k * kJoinThreads + tid, n - 1));
    const float *p[2] = {rows + min(lane, a.parts - 1) * width, rows + min(lane + 64, a.parts - 1) * width};
    const bool here[2] = {lane < a.parts, lane + 64 < a.parts};
    float over = -INFINITY;
    if (a.n_top) {
        const float bound[2] = {here[0] ? p[0][3 + 2 * a.depth] : -INFINITY, here[1] ? p[1][3 + 2 * a.depth] : -INFINITY};
        const int enough = (a.n_top + a.depth - 1) / a.depth;
        if (tid == 0) n_found = 0;
        if (count_above(bound, -INFINITY) >= enough) over = below_nth(bound, enough);
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kMine; k++)
            if (k * kJoinThreads < n && k * kJoinThreads + tid < n && __uint_as_float(mine[k][0]) > over) {
                const int at = atomicAdd(&n_found, 1);  // (in any order: the ranks are the same)
                if (at < kJoinThreads) found[at] = make_uint2(ordered(mine[k][0]), ~mine[k][1]);
            }
        __syncthreads();
        if (64 * wave < n_found && n_found <= kJoinThreads) {
            const uint2 own = tid < n_found ? found[tid] : make_uint2(0, 0);
            const uint64_t key = static_cast<uint64_t>(own.x) << 32 | own.y;
            int rank = 0;
#pragma unroll 8
            for (int i = 0; i < n_found; i++) rank += (static_cast<uint64_t>(found[i].x) << 32 | found[i].y) > key ? 1 : 0;
            if (tid < n_found && rank < 64) sorted[rank] = own;
        }
        __syncthreads();
    }
    if (wave > 0) return;
    const int target = a.target[row];
    const bool in_range = target >= 0 && target < a.vocab;
    const float given = rows[4];
    RowState s;
#pragma unroll
    for (int k = 0; k < 2; k++) {
        RowState o;
        o.most = here[k] ? p[k][0] : kLowest;
        o.sum = here[k] ? p[k][1] : 0.0f;
        o.esum = here[k] ? p[k][2] : 0.0f;
        const float most = fmaxf(s.most, o.most);
        rebase(s, most);
        rebase(o, most);
        s.sum = s.sum + o.sum;
        s.esum = s.esum + o.esum;
        s.above += here[k] ? __builtin_bit_cast(int, p[k][3]) : 0;
    }
    close(s);
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) s.above += __shfl_xor(s.above, o);
    if (a.n_top) {
        if (n_found <= kJoinThreads) {
            s.list = lane < n_found ? sorted[lane].x : 0;
            s.list_low = lane < n_found ? sorted[lane].y : 0;
        } else {  // many alike, or the best side by side: one after the other
            for (int i0 = 0; i0 < n; i0 += 64) {
                const v2u e = entry(min(i0 + lane, n - 1));
                unsigned long long in = __builtin_amdgcn_ballot_w64(i0 + lane < n && __uint_as_float(e[0]) > over);
                while (in) {
                    const int from = __builtin_ctzll(in);
                    in &= in - 1;
                    list_insert(s, ordered(__builtin_amdgcn_readlane(e[0], from)), __builtin_amdgcn_readlane(e[1], from));
                }
                over = fmaxf(over, from_ordered(__builtin_amdgcn_readlane(s.list, a.n_top - 1)));
            }
        }
    }
    write_row<T>(a, row, s, given, in_range, lane);
}

// Parts per row: up to 4096 waves, which the chip holds at once (2048 x 128256 bf16, 20 best: one part a row 130 us, two 113, four 130, every part filling a list of its
// own; 1500 rows: one 130, two 97, four 105; 3000: one 160, two 170), a batch a part at least.  Up to four go into one workgroup, as 1, 2 or 4; four instead of up to
// eight save the second launch (512 x 32000 f32, 5 best: eight 23.8 us, four 18.5; 512 x 128256 bf16, 20 best: 52 either way).  Sixteen waves for a row in one workgroup
// were slower than two launches: a compute unit takes 4 us for sixteen batches, the second launch 3 to 5.
static int score_parts(int64_t n_rows, int64_t vocab) {
    const int64_t batches = (vocab + 1023) / 1024;
    const int parts = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({env_int("CAMELID_HIP_SCORE_WAVES", 4096) / std::max<int64_t>(1, n_rows), batches, kMaxParts})));
    return parts >= 4 && parts <= 8 ? 4 : parts == 3 ? 2 : parts;
}

size_t token_log_probs_workspace(int64_t n_rows, int64_t vocab, int n_top) {
    const int parts = score_parts(n_rows, vocab);
    return parts <= 4 ? 0 : static_cast<size_t>(n_rows) * parts * partial_floats(n_top) * sizeof(float);
}

int launch_token_log_probs(int dtype, const void *logits, int64_t stride, int64_t n_rows, int64_t vocab, const int32_t *target, int n_top, float *log_prob, int32_t *rank, float *entropy,
                           int32_t *top_ids, float *top_log_probs, void *workspace, hipStream_t st) {
    const int64_t batch = dtype == CML_F32 ? 1024 : 2048, batches = (vocab + batch - 1) / batch;
    int parts = static_cast<int>(std::min<int64_t>(score_parts(n_rows, vocab), batches));
    // f32 rows come at memory's rate with fewer waves (20 best of 128256, 1024 rows: two parts 101 us, four 107; 2048: one 186, two 200; 700: two 93, four 77).
    if (dtype == CML_F32 && parts <= 4) parts = static_cast<int>(std::min<int64_t>(parts, std::max<int64_t>(1, 3000 / n_rows)));
    if (parts == 3) parts = 2;
    if (parts > 4 && parts <= 8) parts = 4;
    const int depth = std::max(1, std::min(n_top, (2 * n_top + parts - 1) / parts));
    const ScoreArgs a{logits, target, log_prob, entropy, top_log_probs, rank, top_ids, static_cast<float *>(workspace), stride, n_rows, static_cast<int>(vocab), n_top, parts, depth,
                      n_top ? ((1u << 20) + n_top - 1) / n_top : 0};
    return with_type(dtype, [&](auto t) {
        typedef decltype(t) T;
        const dim3 grid(static_cast<unsigned>((n_rows * a.parts + 3) / 4));
        if (a.parts <= 4) {
            CML_COUNT_LAUNCH("score.rows");
            hipLaunchKernelGGL((token_log_probs_kernel<T, true>), grid, dim3(256), 0, st, a);
        } else {
            CML_COUNT_LAUNCH("score.parts");
            hipLaunchKernelGGL((token_log_probs_kernel<T, false>), grid, dim3(256), 0, st, a);
            hipLaunchKernelGGL(token_log_probs_join_kernel<T>, dim3(static_cast<unsigned>(n_rows)), dim3(kJoinThreads), 0, st, a);
        }
        CML_HIP_TRY(hipGetLastError());
        return CML_OK;
    });
}

}  // namespace cml
