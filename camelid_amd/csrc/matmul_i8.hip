// The int8 product with a scale for every token and every weight row:
//   out[t][r] = rnd((sum_c q[t][c] * w[r][c]) * scales[t] * w_scales[r] + bias[r])
// The sum is an exact 32-bit integer (rows of up to 131071 values: 2^14 * 131071 < 2^31), so no split of the contraction changes a bit.  It is
// widened to f32 (24 bits), scaled in f32 and rounded once to the output's type.
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "gemm_wide.hpp"
#include "typed_rows.hpp"

#pragma clang fp contract(off)

namespace cml {

typedef int v4i_i8 __attribute__((ext_vector_type(4)));

struct MatmulI8 {
    const int8_t *q, *w;
    const float *scales, *w_scales, *bias;
    void *out;
    int64_t q_stride, w_stride, out_stride;
    int n_tokens, rows, cols;
};

// Four neighbouring weight rows of one token.
template <class T>
__device__ __forceinline__ void store_cells(const MatmulI8 &a, int t, int r, const v4i_i8 &acc) {
    if (t >= a.n_tokens) return;
    typename T::Bits *out = static_cast<typename T::Bits *>(a.out) + t * a.out_stride + r;
    const float s = a.scales[t];
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (r + i < a.rows) {
            const float v = static_cast<float>(acc[i]) * s * a.w_scales[r + i];
            store_value<T>(out + i, a.bias ? v + a.bias[r + i] : v);
        }
}

// A pointer that is the same in all lanes, for an operand that has to be in scalar registers.
__device__ __forceinline__ const int8_t *wave_uniform(const int8_t *p) {
    const uint64_t v = reinterpret_cast<uint64_t>(p);
    const uint32_t low = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(v)), high = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(v >> 32));
    return reinterpret_cast<const int8_t *>(static_cast<uint64_t>(high) << 32 | low);
}

// ---- slim tiles -----------------------------------------------------------------------------------------
// For few cells: 16 or 32 weight rows by 16 to 64 tokens a workgroup, so that a product of few cells still has a workgroup for every compute unit, and each of its waves takes lines
// of the rows in turn, by itself: it has LDS of its own, a ring of STAGES lines that requests fill directly, waits for its own requests only, and meets the others where the sums
// are added up.  A request brings whole lines, eight to an instruction: what a unit takes in goes by the lines it has in flight, and in half lines, sixteen to an instruction, straight to
// the lanes that multiply them, it is half as much.  Slot p of a row holds piece p ^ key(row), as below.
//
// Side by side: 16 tokens on 4096 x 14336 13.5 us (in half lines 18.5), on 352 x 15040 8.7 (21); 32 tokens on 4096 x 14336 16.6 (in tiles of 64 x 32 31.6), 64 on 1024 x 4096 4.8 (8.8).
// 1 / 16 / 32 / 64 tokens on 4096 x 14336 with the weight in the last-level cache 11.6 / 12.1 / 12.8 / 15.3 us, from memory 13.8 / 15.0 / 18.1 / 21.7.  What bounds it is the weight's way
// (one token 5.1 and 4.3 TB/s) and for more tokens theirs from the L2.
//
// ANY: rows that start anywhere.  Their lines pass through registers (which takes any address), two of them on their way.  Rows of 4099: one token on 4096 x 4099 5.8 us, 16 6.9,
// in half lines 8.8 and 13.6 (one weight over and over; with three in turn 6.9 and 8.1).
template <class T, int RT, int TT, int WAVES, int STAGES, bool ANY>
__global__ __launch_bounds__(64 * WAVES) void matmul_i8_slim_kernel(MatmulI8 a) {
    constexpr int kRows = 16 * RT, kStage = 16 * (RT + TT) * 128, kFetches = 2 * (RT + TT);
    extern __shared__ uint4 smem[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 15, kq = lane >> 4;
    int row_block, column;
    const int n_row_blocks = (a.rows + kRows - 1) / kRows, n_columns = (a.n_tokens + 16 * TT - 1) / (16 * TT);
    if (a.rows >= a.n_tokens ? !wide_block(blockIdx.x, n_row_blocks, n_columns, row_block, column) : !wide_block(blockIdx.x, n_columns, n_row_blocks, column, row_block)) return;
    const int r0 = row_block * kRows, t0 = column * 16 * TT;
    const int lines = a.cols >> 7, mine = lines > wave ? (lines - wave + WAVES - 1) / WAVES : 0;
    const int8_t *w0 = a.w + static_cast<int64_t>(r0) * a.w_stride + wave * 128, *q0 = a.q + t0 * a.q_stride + wave * 128;
    uint32_t src[kFetches];  // rows 8 f .. 8 f + 7 of the stage: lane 8 r + p brings piece p ^ key(row) of row r
#pragma unroll
    for (int f = 0; f < kFetches; f++) {
        const int at = f * 8 + (lane >> 3);
        const uint32_t piece = ((lane & 7) ^ (at >> 1 & 7)) << 4;
        src[f] = f < 2 * RT ? static_cast<uint32_t>(min(at, a.rows - 1 - r0)) * static_cast<uint32_t>(a.w_stride) + piece
                            : static_cast<uint32_t>(min(at - kRows, a.n_tokens - 1 - t0)) * static_cast<uint32_t>(a.q_stride) + piece;
    }
    typedef int v4i_any __attribute__((ext_vector_type(4), aligned(1)));
    int8_t *lds = reinterpret_cast<int8_t *>(smem) + wave * (STAGES * kStage);
    v4i_i8 acc[RT][TT] = {};
    auto multiply = [&](const v4i_i8 (&w)[RT][2], const v4i_i8 (&q)[TT][2]) __attribute__((always_inline)) {
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int r = 0; r < RT; r++)
#pragma unroll
                for (int t = 0; t < TT; t++) acc[r][t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[r][h], q[t][h], acc[r][t], 0, 0, 0);
    };
    auto multiply_line = [&](int stage) __attribute__((always_inline)) {
        v4i_i8 w[RT][2], q[TT][2];
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int8_t *at = lds + stage * kStage + n * 128 + (((4 * h + kq) ^ (n >> 1)) << 4);
#pragma unroll
            for (int r = 0; r < RT; r++) w[r][h] = *reinterpret_cast<const v4i_i8 *>(at + r * 2048);
#pragma unroll
            for (int t = 0; t < TT; t++) q[t][h] = *reinterpret_cast<const v4i_i8 *>(at + (RT + t) * 2048);
        }
        multiply(w, q);
    };
    if (mine > 0) {
        if constexpr (ANY) {
            // lines pass through registers, two of them on their way
            v4i_i8 one[kFetches], two[kFetches];
            auto load = [&](v4i_i8 (&to)[kFetches], int i) __attribute__((always_inline)) {
                const int64_t at = static_cast<int64_t>(min(i, mine - 1)) * (WAVES * 128);
#pragma unroll
                for (int f = 0; f < kFetches; f++) to[f] = *reinterpret_cast<const v4i_any *>((f < 2 * RT ? w0 : q0) + at + src[f]);
            };
            auto line = [&](v4i_i8 (&of)[kFetches], int i) __attribute__((always_inline)) {
#pragma unroll
                for (int f = 0; f < kFetches; f++) *reinterpret_cast<v4i_i8 *>(lds + f * 1024 + lane * 16) = of[f];
                load(of, i + 2);
                __builtin_amdgcn_wave_barrier();
                multiply_line(0);
                __builtin_amdgcn_wave_barrier();
            };
            load(one, 0);
            load(two, 1);
            int i = 0;
            for (; i + 1 < mine; i += 2) {
                line(one, i);
                line(two, i + 1);
            }
            if (i < mine) line(one, i);
        } else {
            const uint32_t lds0 = lds_address(smem) + wave * (STAGES * kStage);
            auto fetch = [&](int i, int stage) __attribute__((always_inline)) {
                const int64_t at = static_cast<int64_t>(min(i, mine - 1)) * (WAVES * 128);
#pragma unroll
                for (int f = 0; f < kFetches; f++) wide_dma16(lds0 + stage * kStage + f * 1024, wave_uniform((f < 2 * RT ? w0 : q0) + at), src[f]);
            };
#pragma unroll
            for (int k = 0; k < STAGES - 1; k++) fetch(k, k);
            int stage = 0, into = STAGES - 1;
            for (int i = 0; i < mine; i++) {
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // what was read last may be overwritten
                fetch(i + STAGES - 1, into);                        // (past the end the last line again: the number of requests in flight stays the same)
                wide_wait<(STAGES - 1) * kFetches>();
                multiply_line(stage);
                into = stage;
                stage = stage == STAGES - 1 ? 0 : stage + 1;
            }
            wide_wait<0>();
        }
    }
    if ((a.cols & 127) && lines % WAVES == wave) {  // the rest of the rows, zeros behind their ends
        auto piece = [&](const int8_t *p, int c) {
            v4i_i8 v = {};
            if (c + 16 <= a.cols) return static_cast<v4i_i8>(*reinterpret_cast<const v4i_any *>(p + c));
            for (int j = 0; c + j < a.cols; j++) v[j >> 2] |= static_cast<int>(static_cast<uint32_t>(static_cast<uint8_t>(p[c + j])) << (8 * (j & 3)));
            return v;
        };
        v4i_i8 w[RT][2], q[TT][2];
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int c = lines * 128 + (4 * h + kq) * 16;
#pragma unroll
            for (int r = 0; r < RT; r++) w[r][h] = piece(a.w + static_cast<int64_t>(min(r0 + 16 * r + n, a.rows - 1)) * a.w_stride, c);
#pragma unroll
            for (int t = 0; t < TT; t++) q[t][h] = piece(a.q + static_cast<int64_t>(min(t0 + 16 * t + n, a.n_tokens - 1)) * a.q_stride, c);
        }
        multiply(w, q);
    }
    __syncthreads();  // (LDS changes its use)
    v4i_i8 *part = reinterpret_cast<v4i_i8 *>(smem);
#pragma unroll
    for (int r = 0; r < RT; r++)
#pragma unroll
        for (int t = 0; t < TT; t++) part[((r * TT + t) * WAVES + wave) * 64 + lane] = acc[r][t];
    __syncthreads();
    for (int c = wave; c < RT * TT; c += WAVES) {
        v4i_i8 sum = {};
#pragma unroll
        for (int k = 0; k < WAVES; k++) sum += part[(c * WAVES + k) * 64 + lane];
        store_cells<T>(a, t0 + 16 * (c % TT) + n, r0 + 16 * (c / TT) + 4 * kq, sum);
    }
}

// ---- tiles --------------------------------------------------------------------------------------------
// Rows on 16-byte boundaries.  WR x WT waves of MT x NT tiles of 32 x 32 cells; a step is 128 values of the contraction: whole lines of both operands
// go to LDS without passing through registers, into the oldest of STAGES steps as soon as it has been read.  Slot p of an LDS row (16 bytes) holds piece p ^ key(row), so that the eight rows that
// eight neighbouring lanes read lie in different banks.
//
// The instruction's 32 rows are the tile's in another order: a lane ends up with 16 neighbouring weight rows of its token and stores them whole.
//
// 37 tokens on 128256 x 2048: 54 us, the weight and the logits at 5.2 TB/s.  4096 x 14336 x 4096 (the walk): 217 - 225 us, 2.2 POPS; the matrix cores execute 56 % of the busy
// cycles, LDS conflicts are gone, and the clock is the limit: under this load it falls from 2.4 to 1.8 GHz (8192 x 8192 x 8192: 455 - 463 us, of zeros 335).
typedef int v16i_i8 __attribute__((ext_vector_type(16)));

struct TileGrid {
    int n_row_blocks, n_token_blocks, group;
};

// The at-th tile in the order of bands of `group` token blocks, row block after row block: neighbours share rows of both operands.  Consecutive workgroup
// ids go to the eight XCDs in turn; each XCD gets a run of its own of that order, so that what its tiles share comes through its L2 once.
__device__ __forceinline__ void tile_of(const TileGrid &g, int at, int &row_block, int &token_block, int &wide) {
    const int band = at / (g.group * g.n_row_blocks), in = at - band * g.group * g.n_row_blocks;
    wide = min(g.group, g.n_token_blocks - band * g.group);
    row_block = in / wide;
    token_block = band * g.group + in - row_block * wide;
}

// One tile's work by a workgroup of WR x WT waves.  SPLIT: the tile has 1 / SPLIT of the rows.  FULL: every row and token of the tile is there.
template <class T, int WR, int WT, int MT, int NT, int STAGES, bool ONCE, bool FULL>
struct TileWork {
    static constexpr int KB = 128;  // values of the contraction a step: a whole line of a row
    static constexpr int kWaves = WR * WT, kThreads = 64 * kWaves, kRows = WR * MT * 32, kTokens = WT * NT * 32;
    static constexpr int kPass = kThreads / 8;  // rows that one pass of the workgroup fetches
    static constexpr int kStage = (kRows + kTokens) * KB, kFetches = (kRows + kTokens) / kPass, kWeightFetches = kRows / kPass;
    static constexpr int kTouch = FULL, kParts = KB / 32;
    static constexpr int kScales = STAGES * kStage + kTouch * kWaves * 256, kLds = kScales + 8 * kRows;  // stages, what touch() fills, scales and bias of the rows
    static_assert((kRows + kTokens) % kPass == 0 && kRows % kPass == 0, "whole passes of the workgroup");

    const MatmulI8 &a;
    const int8_t *lds;
    uint32_t lds0;
    int tid, lane, wave, wr, wt, m, half, row_a, n_steps;
    int r0, t0;                 // of the tile that is fetched
    uint32_t src[FULL ? 2 : kFetches];
    const int8_t *touched;
    bool touches;
    uint32_t at_a, at_b;
    v16i_i8 acc[MT][NT];
    v4i_i8 fa[2][MT], fb[2][NT];

    // (sixteen lanes read at a time; 64 banks are two rows of 128 bytes)
    static __device__ __forceinline__ int key_w(int row) { return (row >> 1 & 3) | (row >> 2 & 4); }
    static __device__ __forceinline__ int key_q(int row) { return row >> 1 & 7; }

    __device__ __forceinline__ TileWork(const MatmulI8 &args, uint4 *smem) : a(args) {
        lds = reinterpret_cast<const int8_t *>(smem);
        lds0 = lds_address(smem);
        tid = threadIdx.x;
        lane = tid & 63;
        wave = __builtin_amdgcn_readfirstlane(tid >> 6);
        wr = wave / WT;
        wt = wave - wr * WT;
        m = lane & 31;
        half = lane >> 5;
        row_a = (m & 3) | (m >> 1 & 12) | (m << 2 & 16);  // instruction row 8a + 4b + c is the tile's 16b + 4a + c
        n_steps = a.cols / KB;
        at_a = (wr * MT * 32 + row_a) * KB + ((half ^ key_w(row_a)) << 4);  // of part 0; part s has piece 2 s + half: the address exclusive-or 32 s
        at_b = (kRows + wt * NT * 32 + m) * KB + ((half ^ key_q(m)) << 4);
    }

    // Pass k of the workgroup takes LDS rows k * kPass ..; the weight's rows first, then the tokens'.  Rows past the end repeat the last one.
    template <int SPLIT>
    __device__ __forceinline__ void aim(int row, int token, int row_share, int wide, int token_share) {
        constexpr int kMine = kRows / SPLIT;
        r0 = row;
        t0 = token;
        int tid = this->tid;
        asm volatile("" : "+v"(tid));  // (as in store)
        const int f_row = tid >> 3, f_slot = tid & 7;
        if constexpr (FULL) {  // (the keys of rows kPass apart are the same: one offset, and a base for every pass)
            static_assert(kPass % 32 == 0, "keys");
            src[0] = f_row * static_cast<uint32_t>(a.w_stride) + ((f_slot ^ key_w(f_row)) << 4);
            src[1] = f_row * static_cast<uint32_t>(a.q_stride) + ((f_slot ^ key_q(f_row)) << 4);
        } else
#pragma unroll
        for (int k = 0; k < kFetches; k++) {
            const int at = k * kPass + f_row, t = at - kRows;
            src[k] = k < kWeightFetches ? static_cast<uint32_t>(min(at, a.rows - 1 - r0)) * static_cast<uint32_t>(a.w_stride) + ((f_slot ^ key_w(at)) << 4)
                                        : static_cast<uint32_t>(min(t, a.n_tokens - 1 - t0)) * static_cast<uint32_t>(a.q_stride) + ((f_slot ^ key_q(t)) << 4);
        }
        if constexpr (kTouch) {
            // Lines of a later step into the L2: 32 compute units share it, `wide` of them a tile's weight rows and the others of a column its tokens;
            // each asks for its part of both, four bytes a line, into LDS that nobody reads.
            const int share_w = (kMine + wide - 1) / wide, per_w = (share_w + kWaves - 1) / kWaves, deep = 32 / wide, share_q = (kTokens + deep - 1) / deep, per_q = (share_q + kWaves - 1) / kWaves;
            const int touch_w = row_share * share_w + wave * per_w + lane, touch_q = token_share % deep * share_q + wave * per_q + lane - per_w;
            touches = lane < per_w + per_q;
            const int8_t *w0 = weights(), *q0 = tokens();
            touched = lane < per_w ? w0 + min(touch_w, min(kMine, a.rows - r0) - 1) * a.w_stride : q0 + min(max(touch_q, 0), min(kTokens, a.n_tokens - t0) - 1) * a.q_stride;
        }
    }
    // First bytes of the tile's weight rows and tokens, in scalar registers.
    __device__ __forceinline__ const int8_t *weights() const { return a.w + static_cast<int64_t>(__builtin_amdgcn_readfirstlane(r0)) * a.w_stride; }
    __device__ __forceinline__ const int8_t *tokens() const { return a.q + static_cast<int64_t>(__builtin_amdgcn_readfirstlane(t0)) * a.q_stride; }
    __device__ __forceinline__ void fetch(const int8_t *w0, const int8_t *q0, int k, int step, int stage) {
        const uint32_t to = (lds0 + stage * kStage + k * (16 * kThreads) + wave * 1024);
        const bool weight = k < kWeightFetches;
        const int8_t *from = (weight ? w0 : q0) + step * KB;
        if constexpr (FULL) from += static_cast<int64_t>(weight ? k : k - kWeightFetches) * kPass * (weight ? a.w_stride : a.q_stride);
        const uint32_t off = src[FULL ? (weight ? 0 : 1) : k];
        if (ONCE && weight) wide_dma16_once(to, wave_uniform(from), off);
        else wide_dma16(to, wave_uniform(from), off);
    }
    __device__ __forceinline__ void touch(int step) {
        if constexpr (kTouch) {
            const int8_t *at = touched + step * KB;
            const uint32_t to = __builtin_amdgcn_readfirstlane(lds0 + STAGES * kStage + wave * 256);
            // (m0 is set where it is used: between two statements it could become another)
            if (touches) asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(to), "v"(at) : "memory", "m0");
        }
    }
    template <int SPLIT>
    static constexpr bool fetched(int k) { return k >= kWeightFetches || k < kWeightFetches / SPLIT; }
    template <int SPLIT>
    static constexpr int fetches() { return kWeightFetches / SPLIT + kFetches - kWeightFetches; }
    template <int SPLIT>
    __device__ __forceinline__ void start() {
        if (n_steps == 0) return;
        const int8_t *w0 = weights(), *q0 = tokens();
#pragma unroll
        for (int k = 0; k < STAGES - 1; k++)
#pragma unroll
            for (int f = 0; f < kFetches; f++)
                if (fetched<SPLIT>(f)) fetch(w0, q0, f, min(k, n_steps - 1), k);
        touch(min(STAGES, n_steps - 1));
    }
    // The last step where it is not whole: through registers, zeros behind the rows' ends; two to four pieces on their way at a time (2899 x 8126 x 960: one 48 us, 45).
    template <int SPLIT>
    __device__ __forceinline__ void fetch_rest(uint4 *smem) {
        constexpr int kBatch = FULL ? 2 : kFetches % 4 == 0 ? 4 : 3;
        static_assert(kFetches % kBatch == 0, "batches");
        const int8_t *w0 = weights(), *q0 = tokens();
#pragma unroll 1
        for (int k0 = 0; k0 < kFetches; k0 += kBatch) {
            uint4 v[kBatch];
            const int8_t *from[kBatch];
            int c[kBatch];
#pragma unroll
            for (int u = 0; u < kBatch; u++) {
                const int at = (k0 + u) * kPass + (tid >> 3), t = at - kRows;
                const int piece = at < kRows ? (tid & 7) ^ key_w(at) : (tid & 7) ^ key_q(t);
                const int8_t *p = at < kRows ? w0 + min(at, a.rows - 1 - r0) * a.w_stride : q0 + min(t, a.n_tokens - 1 - t0) * a.q_stride;
                c[u] = n_steps * KB + piece * 16;
                from[u] = p + c[u];
                v[u] = make_uint4(0, 0, 0, 0);
                if (fetched<SPLIT>(k0 + u) && c[u] + 16 <= a.cols) v[u] = ldg16(from[u]);
            }
            if (a.cols & 15)
#pragma unroll
                for (int u = 0; u < kBatch; u++)
                    if (fetched<SPLIT>(k0 + u) && c[u] < a.cols && c[u] + 16 > a.cols) {
                        uint32_t b[4] = {0, 0, 0, 0};
                        for (int j = 0; c[u] + j < a.cols; j++) b[j >> 2] |= static_cast<uint32_t>(static_cast<uint8_t>(from[u][j])) << (8 * (j & 3));
                        v[u] = make_uint4(b[0], b[1], b[2], b[3]);
                    }
#pragma unroll
            for (int u = 0; u < kBatch; u++)
                if (fetched<SPLIT>(k0 + u)) smem[(k0 + u) * kThreads + tid] = v[u];
        }
    }

    // Operands of a 32-value part of the step are read while the matrix cores work on the part before: two sets of registers, in turn.
    template <int SPLIT>
    __device__ __forceinline__ void read(int stage, int s) {
        const int8_t *pa = lds + stage * kStage + ((at_a ^ (32 * s)) - wr * (MT - MT / SPLIT) * 32 * KB), *pb = lds + stage * kStage + (at_b ^ (32 * s));
#pragma unroll
        for (int i = 0; i < MT / SPLIT; i++) fa[s & 1][i] = *reinterpret_cast<const v4i_i8 *>(pa + i * 32 * KB);
#pragma unroll
        for (int j = 0; j < NT; j++) fb[s & 1][j] = *reinterpret_cast<const v4i_i8 *>(pb + j * 32 * KB);
        __builtin_amdgcn_sched_barrier(0);
    }
    // Requests go out one at a time between the matrix instructions (a wave that issues many in a row waits for the address unit): request f behind
    // instruction f * span / fetches.
    template <int SPLIT, bool FETCH>
    __device__ __forceinline__ void multiply(const int8_t *w0, const int8_t *q0, int s, int step, int stage) {
        constexpr int kN = fetches<SPLIT>(), kSlots = MT / SPLIT * NT * (kParts - 1), kSpan = kSlots < 2 * kN ? kSlots : 2 * kN;
#pragma unroll
        for (int i = 0; i < MT / SPLIT; i++)
#pragma unroll
            for (int j = 0; j < NT; j++) {
                acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fa[s & 1][i], fb[s & 1][j], acc[i][j], 0, 0, 0);
                const int at = (s * (MT / SPLIT) + i) * NT + j;
                if (FETCH && at < kSpan) {
                    __builtin_amdgcn_sched_barrier(0);
                    int n = 0;
#pragma unroll
                    for (int f = 0; f < kFetches; f++)
                        if (fetched<SPLIT>(f)) {
                            if (n * kSpan / kN == at) fetch(w0, q0, f, step, stage);
                            n++;
                        }
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
        __builtin_amdgcn_sched_barrier(0);
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < MT; i++)
#pragma unroll
            for (int j = 0; j < NT; j++) acc[i][j] = v16i_i8{};
    }
    // The sums of the tile that aim() and start() began.
    template <int SPLIT>
    __device__ __forceinline__ void sums(uint4 *smem) {
        constexpr int kN = fetches<SPLIT>();
        const int8_t *w0 = weights(), *q0 = tokens();
        clear();
        if (n_steps > 0) {
            wide_wait<(STAGES - 2) * kN + kTouch>();
            wide_barrier();
            int stage = 0, into = STAGES - 1;  // the stage that was read last is filled next
            read<SPLIT>(0, 0);
            for (int step = 0; step < n_steps; step++) {
                const int ahead = min(step + STAGES - 1, n_steps - 1);  // (past the end the last step again: the number of requests in flight stays the same)
#pragma unroll
                for (int s = 0; s + 1 < kParts; s++) {
                    read<SPLIT>(stage, s + 1);
                    multiply<SPLIT, true>(w0, q0, s, ahead, into);
                }
                touch(min(step + STAGES + 1, n_steps - 1));
                into = stage;
                stage = stage == STAGES - 1 ? 0 : stage + 1;
                wide_wait<(STAGES - 2) * (kN + kTouch) + kTouch>();
                wide_barrier();  // the next step is there for every wave, and every wave has read this one
                read<SPLIT>(stage, 0);
                multiply<SPLIT, false>(w0, q0, kParts - 1, 0, 0);
            }
            wide_wait<0>();
        }
        wide_barrier();  // (what was asked for past the end has come, for every wave: LDS is free)
        if (a.cols % KB) {
            fetch_rest<SPLIT>(smem);
            wide_barrier();
#pragma unroll
            for (int s = 0; s < kParts; s++) {
                read<SPLIT>(0, s);
                multiply<SPLIT, false>(w0, q0, s, 0, 0);
            }
            wide_barrier();
        }
    }
    // A lane has 16 neighbouring rows of one token: stored so, a wave would write 16 bytes here and there (256 x 256 cells 10 us).  They change places in LDS, each
    // wave's in its own 8 KB of the second stage, 32 tokens by up to 256 bytes at a time, and leave as whole runs.  Slots are exclusive-ored here too.
    // STREAM: past the caches.
    template <int SPLIT, bool STREAM = false>
    __device__ __forceinline__ void store(uint4 *smem, int row, int token) {
        row = __builtin_amdgcn_readfirstlane(row);
        token = __builtin_amdgcn_readfirstlane(token);
        typedef typename T::Bits Bits;
        // (what follows depends on this copy: otherwise its addresses are kept in registers through the sums of every tile)
        int lane = this->lane;
        asm volatile("" : "+v"(lane));
        const int m = lane & 31, half = lane >> 5;
        constexpr int kMine = MT / SPLIT, kPhase = kMine * 32 * static_cast<int>(sizeof(Bits)) > 256 ? 8 / static_cast<int>(sizeof(Bits)) : kMine;  // row tiles at a time
        constexpr int kSlots = kPhase * 32 * static_cast<int>(sizeof(Bits)) / 16, kPer = 16 / static_cast<int>(sizeof(Bits));
        static_assert(STAGES * kStage - kStage >= kWaves * 32 * kSlots * 16, "LDS behind the first stage");
        uint4 *mine = smem + kStage / 16 + wave * (32 * kSlots);
        float *scales = reinterpret_cast<float *>(smem + kScales / 16);
        for (int r = tid; r < kRows / SPLIT; r += kThreads) {
            scales[r] = a.w_scales[min(row + r, a.rows - 1)];
            scales[kRows + r] = a.bias ? a.bias[min(row + r, a.rows - 1)] : 0.0f;
        }
        wide_barrier();
        auto swap = [](int t, int slot) { return t * kSlots + (slot ^ (kSlots == 16 ? t & 15 : kSlots == 8 ? t >> 1 & 7 : t >> 2 & 3)); };
#pragma unroll
        for (int i0 = 0; i0 < kMine; i0 += kPhase) {
#pragma unroll
            for (int j = 0; j < NT; j++) {
                const int t0 = token + (wt * NT + j) * 32;
                const float s = a.scales[FULL ? t0 + m : min(t0 + m, a.n_tokens - 1)];
#pragma unroll
                for (int i = 0; i < kPhase; i++) {
                    const int r = (wr * kMine + i0 + i) * 32 + 16 * half;
                    float v[16];
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const float4 f = *reinterpret_cast<const float4 *>(scales + r + 4 * k);
                        v[4 * k] = static_cast<float>(acc[i0 + i][j][4 * k]) * s * f.x;
                        v[4 * k + 1] = static_cast<float>(acc[i0 + i][j][4 * k + 1]) * s * f.y;
                        v[4 * k + 2] = static_cast<float>(acc[i0 + i][j][4 * k + 2]) * s * f.z;
                        v[4 * k + 3] = static_cast<float>(acc[i0 + i][j][4 * k + 3]) * s * f.w;
                    }
                    if (a.bias)
#pragma unroll
                        for (int k = 0; k < 4; k++) {
                            const float4 f = *reinterpret_cast<const float4 *>(scales + kRows + r + 4 * k);
                            v[4 * k] = v[4 * k] + f.x;
                            v[4 * k + 1] = v[4 * k + 1] + f.y;
                            v[4 * k + 2] = v[4 * k + 2] + f.z;
                            v[4 * k + 3] = v[4 * k + 3] + f.w;
                        }
#pragma unroll
                    for (int k = 0; k < 16 / kPer; k++) {
                        uint4 packed;
                        if constexpr (sizeof(Bits) == 4)
                            packed = make_uint4(__float_as_uint(v[4 * k]), __float_as_uint(v[4 * k + 1]), __float_as_uint(v[4 * k + 2]), __float_as_uint(v[4 * k + 3]));
                        else
                            packed = make_uint4(T::narrow(v[8 * k]) | T::narrow(v[8 * k + 1]) << 16, T::narrow(v[8 * k + 2]) | T::narrow(v[8 * k + 3]) << 16,
                                                T::narrow(v[8 * k + 4]) | T::narrow(v[8 * k + 5]) << 16, T::narrow(v[8 * k + 6]) | T::narrow(v[8 * k + 7]) << 16);
                        mine[swap(m, (2 * i + half) * (16 / kPer) + k)] = packed;
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
                const int r = row + (wr * kMine + i0) * 32;
#pragma unroll
                for (int q = 0; q < kSlots / 2; q++) {
                    const int at = q * 64 + lane, t = at / kSlots, slot = at % kSlots, rr = r + slot * kPer;
                    const uint4 v = mine[swap(t, slot)];
                    if (!FULL && (t0 + t >= a.n_tokens || rr >= a.rows)) continue;
                    Bits *out = static_cast<Bits *>(a.out) + (t0 + t) * a.out_stride + rr;
                    if (FULL || rr + kPer <= a.rows) {
                        typedef uint32_t v4u __attribute__((ext_vector_type(4), aligned(2)));
                        if constexpr (STREAM) __builtin_nontemporal_store(v4u{v.x, v.y, v.z, v.w}, reinterpret_cast<v4u *>(out));
                        else *reinterpret_cast<v4u *>(out) = v4u{v.x, v.y, v.z, v.w};
                    } else {
                        const uint32_t word[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                        for (int e = 0; e < kPer; e++)
                            if (rr + e < a.rows) out[e] = sizeof(Bits) == 4 ? __builtin_bit_cast(Bits, static_cast<std::conditional_t<sizeof(Bits) == 4, uint32_t, uint16_t>>(word[e])) : __builtin_bit_cast(Bits, static_cast<std::conditional_t<sizeof(Bits) == 4, uint32_t, uint16_t>>(word[e / 2] >> (16 * (e & 1))));
                    }
                }
            }
        }
    }
};

// A workgroup a tile.
template <class T, int WR, int WT, int MT, int NT, int STAGES, int PER_CU, bool ONCE>
__global__ __launch_bounds__(64 * WR * WT, WR * WT * PER_CU / 4) void matmul_i8_tile_kernel(MatmulI8 a, TileGrid grid) {
    extern __shared__ uint4 smem[];
    TileWork<T, WR, WT, MT, NT, STAGES, ONCE, false> work(a, smem);
    const int total = grid.n_row_blocks * grid.n_token_blocks, per = total >> 3, more = total & 7, xcd = blockIdx.x & 7;
    int row_block, token_block, wide;
    tile_of(grid, xcd * per + min(xcd, more) + (blockIdx.x >> 3), row_block, token_block, wide);
    const int row = row_block * work.kRows, token = token_block * work.kTokens;
    work.template aim<1>(row, token, token_block % wide, wide, row_block);
    work.template start<1>();
    work.template sums<1>(smem);
    work.template store<1>(smem, row, token);
}

// Rows that start anywhere: a workgroup a tile, through registers (which takes any address), two steps ahead, zeros behind the rows' ends.  4096 x 4096 x 4096 in rows of 4099: 125 us,
// on 16-byte boundaries 66: registers hold what is on its way, so less of it is.
template <class T, int MT>
__global__ __launch_bounds__(256) void matmul_i8_staged_kernel(MatmulI8 a, TileGrid grid) {
    extern __shared__ uint4 smem[];
    typedef TileWork<T, 2, 2, MT, MT, 2, false, false> Work;
    Work work(a, smem);
    constexpr int kFetches = Work::kFetches;
    const int total = grid.n_row_blocks * grid.n_token_blocks, per = total >> 3, more = total & 7, xcd = blockIdx.x & 7;
    int row_block, token_block, wide;
    tile_of(grid, xcd * per + min(xcd, more) + (blockIdx.x >> 3), row_block, token_block, wide);
    const int row = row_block * Work::kRows, token = token_block * Work::kTokens, n_steps = (a.cols + 127) >> 7;
    const int tid = threadIdx.x, slot = tid & 7;
    const int8_t *from[kFetches];
    int piece[kFetches];
#pragma unroll
    for (int k = 0; k < kFetches; k++) {
        const int at = k * Work::kPass + (tid >> 3), t = at - Work::kRows;
        piece[k] = 16 * (k < Work::kWeightFetches ? slot ^ Work::key_w(at) : slot ^ Work::key_q(t));
        from[k] = (k < Work::kWeightFetches ? a.w + min(row + at, a.rows - 1) * a.w_stride : a.q + min(token + t, a.n_tokens - 1) * a.q_stride) + piece[k];
    }
    auto request = [&](int step, uint4 (&v)[kFetches]) __attribute__((always_inline)) {
        typedef uint32_t v4u __attribute__((ext_vector_type(4), aligned(1)));
        if ((step + 1) * 128 <= a.cols) {
#pragma unroll
            for (int k = 0; k < kFetches; k++) {
                const v4u w = *reinterpret_cast<const v4u *>(from[k] + step * 128);
                v[k] = make_uint4(w.x, w.y, w.z, w.w);
            }
            return;
        }
#pragma unroll
        for (int k = 0; k < kFetches; k++) {
            const int8_t *p = from[k] + step * 128;
            const int c = step * 128 + piece[k];
            v[k] = make_uint4(0, 0, 0, 0);
            if (c + 16 <= a.cols) {
                const v4u w = *reinterpret_cast<const v4u *>(p);
                v[k] = make_uint4(w.x, w.y, w.z, w.w);
            } else if (c < a.cols) {
                uint32_t b[4] = {0, 0, 0, 0};
                for (int j = 0; c + j < a.cols; j++) b[j >> 2] |= static_cast<uint32_t>(static_cast<uint8_t>(p[j])) << (8 * (j & 3));
                v[k] = make_uint4(b[0], b[1], b[2], b[3]);
            }
        }
    };
    uint4 even[kFetches], odd[kFetches];
    work.clear();
    auto step = [&](int s, uint4 (&v)[kFetches]) __attribute__((always_inline)) {
#pragma unroll
        for (int k = 0; k < kFetches; k++) smem[((s & 1) * Work::kStage + k * 16 * Work::kThreads) / 16 + tid] = v[k];
        if (s + 2 < n_steps) request(s + 2, v);
        wide_barrier();  // (one a step: the other stage is not written again before every wave is through this step's)
        work.template read<1>(s & 1, 0);
#pragma unroll
        for (int part = 0; part < Work::kParts; part++) {
            if (part + 1 < Work::kParts) work.template read<1>(s & 1, part + 1);
            work.template multiply<1, false>(nullptr, nullptr, part, 0, 0);
        }
    };
    request(0, even);
    if (n_steps > 1) request(1, odd);
    for (int s = 0; s < n_steps; s += 2) {
        step(s, even);
        if (s + 1 < n_steps) step(s + 1, odd);
    }
    wide_barrier();
    work.template store<1>(smem, row, token);
}

// A workgroup a compute unit, 32 an XCD: each walks the tiles of its XCD's run 32 apart, and asks for the next tile's first step before it stores the one
// it has.  The tiles that are left when all 32 can no longer have a whole one are cut into halves or quarters of their rows where that gives every
// unit some (896 tiles, 4096 tokens on 14336 rows: the time of 3.5 tiles instead of 4).  The last tiles of a side that is no whole number of them reach back
// into their neighbours: cells that two workgroups write get the same bits.
template <class T, int WR, int WT, int MT, int NT, bool STREAM>
__global__ __launch_bounds__(64 * WR * WT, WR * WT / 4) void matmul_i8_walk_kernel(MatmulI8 a, TileGrid grid) {
    extern __shared__ uint4 smem[];
    TileWork<T, WR, WT, MT, NT, 2, false, true> work(a, smem);
    constexpr int kRows = work.kRows, kTokens = work.kTokens;
    const int total = grid.n_row_blocks * grid.n_token_blocks, per = total >> 3, more = total & 7, xcd = blockIdx.x & 7, unit = blockIdx.x >> 3;
    const int first = xcd * per + min(xcd, more), n = per + (xcd < more ? 1 : 0);
    const int rounds = n >> 5, left = n & 31, split = left == 0 || left > 16 ? 1 : left > 8 ? 2 : 4;
    // This unit's items: whole tiles and at most one part.  Every other unit takes its part first, so that not all of them come to their stores at the
    // same time.
    const bool part = split > 1 && unit < left * split, part_first = part && (unit & 1) != 0;
    const int wholes = rounds + (split == 1 && unit < left ? 1 : 0), items = wholes + (part ? 1 : 0);
    int row = 0, token = 0;
    auto is_part = [&](int item) __attribute__((always_inline)) { return part && item == (part_first ? 0 : wholes); };
    auto begin = [&](int item) __attribute__((always_inline)) {
        int row_block, token_block, wide;
        if (!is_part(item)) {
            tile_of(grid, first + (item - (part_first ? 1 : 0)) * 32 + unit, row_block, token_block, wide);
            row = min(row_block * kRows, a.rows - kRows);
            token = min(token_block * kTokens, a.n_tokens - kTokens);
            work.template aim<1>(row, token, token_block % wide, wide, row_block);
            work.template start<1>();
        } else {
            tile_of(grid, first + rounds * 32 + unit / split, row_block, token_block, wide);
            row = min(row_block * kRows, a.rows - kRows) + unit % split * (kRows / split);
            token = min(token_block * kTokens, a.n_tokens - kTokens);
            if (split == 2) {
                work.template aim<2>(row, token, 0, 1, 0);
                work.template start<2>();
            } else {
                work.template aim<4>(row, token, 0, 1, 0);
                work.template start<4>();
            }
        }
    };
    if (items > 0) begin(0);
#pragma unroll 1
    for (int item = 0; item < items; item++) {
        const int cut = is_part(item) ? split : 1, r = row, t = token;
        auto run = [&](auto parts) __attribute__((always_inline)) {
            constexpr int kParts = decltype(parts)::value;
            work.template sums<kParts>(smem);
            if (item + 1 < items) begin(item + 1);
            work.template store<kParts, STREAM>(smem, r, t);
        };
        if (cut == 1) run(std::integral_constant<int, 1>{});
        else if (cut == 2) run(std::integral_constant<int, 2>{});
        else run(std::integral_constant<int, 4>{});
    }
}

template <class K>
static int allow_lds(K kernel, size_t bytes, std::atomic<bool> &raised) {
    if (bytes > 64 * 1024 && !raised.load(std::memory_order_acquire)) {  // (a launch may use that much without asking)
        CML_HIP_TRY(hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes)));
        raised.store(true, std::memory_order_release);
    }
    return CML_OK;
}

inline TileGrid tile_grid(const MatmulI8 &a, int rows, int tokens) {
    const int n = (a.n_tokens + tokens - 1) / tokens;
    return TileGrid{(a.rows + rows - 1) / rows, n, std::min(4, n)};
}

// Calls launch(part) for as many of the tokens at a time, in whole tiles of `tokens`, as a launch has workgroups of `threads` for; row_blocks of them take a token block
// (and seven blocks more, where a grid has them in eights).
template <class T, class F>
static int over_tokens(const MatmulI8 &a, int64_t row_blocks, int tokens, int threads, F launch) {
    const int64_t most = std::max<int64_t>(1, most_workgroups(threads) / row_blocks - 7) * tokens;
    for (int64_t first = 0; first < a.n_tokens; first += most) {
        MatmulI8 part = a;
        part.q = a.q + first * a.q_stride;
        part.scales = a.scales + first;
        part.out = static_cast<typename T::Bits *>(a.out) + first * a.out_stride;
        part.n_tokens = static_cast<int>(std::min<int64_t>(most, a.n_tokens - first));
        launch(part);
        CML_HIP_TRY(hipGetLastError());
    }
    return CML_OK;
}

template <class T, int WR, int WT, int MT, int NT, int STAGES, int PER_CU, bool ONCE = false>
static int launch_tile(const MatmulI8 &a, hipStream_t st) {
    typedef TileWork<T, WR, WT, MT, NT, STAGES, ONCE, false> Work;
    static_assert(Work::kLds * PER_CU <= 160 * 1024, "LDS");
    const auto kernel = matmul_i8_tile_kernel<T, WR, WT, MT, NT, STAGES, PER_CU, ONCE>;
    static std::atomic<bool> raised{false};
    if (int rc = allow_lds(kernel, Work::kLds, raised)) return rc;
    return over_tokens<T>(a, (a.rows + Work::kRows - 1) / Work::kRows, Work::kTokens, Work::kThreads, [&](const MatmulI8 &part) {
        const TileGrid grid = tile_grid(part, Work::kRows, Work::kTokens);
        CML_COUNT_LAUNCH(ONCE ? "i8.matmul.tile.once" : "i8.matmul.tile");
        hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(grid.n_row_blocks * grid.n_token_blocks)), dim3(Work::kThreads), Work::kLds, st, part, grid);
    });
}

template <class T, int RT, int TT, int WAVES, int STAGES, bool ANY>
static int launch_slim(const MatmulI8 &a, hipStream_t st) {
    constexpr int kLds = WAVES * STAGES * 16 * (RT + TT) * 128;
    static_assert(kLds <= 160 * 1024 && kLds >= RT * TT * WAVES * 1024, "LDS");
    const int n_row_blocks = (a.rows + 16 * RT - 1) / (16 * RT);
    const auto kernel = matmul_i8_slim_kernel<T, RT, TT, WAVES, STAGES, ANY>;
    static std::atomic<bool> raised{false};
    if (int rc = allow_lds(kernel, kLds, raised)) return rc;
    return over_tokens<T>(a, n_row_blocks + 7, 16 * TT, 64 * WAVES, [&](const MatmulI8 &part) {
        const int n_columns = (part.n_tokens + 16 * TT - 1) / (16 * TT);
        CML_COUNT_LAUNCH(ANY ? "i8.matmul.slim.any" : "i8.matmul.slim");
        hipLaunchKernelGGL(kernel, dim3(part.rows >= part.n_tokens ? wide_grid(n_row_blocks, n_columns) : wide_grid(n_columns, n_row_blocks)), dim3(64 * WAVES), kLds, st, part);
    });
}

template <class T, int MT>
static int launch_staged(const MatmulI8 &a, hipStream_t st) {
    typedef TileWork<T, 2, 2, MT, MT, 2, false, false> Work;
    const auto kernel = matmul_i8_staged_kernel<T, MT>;
    static std::atomic<bool> raised{false};
    if (int rc = allow_lds(kernel, Work::kLds, raised)) return rc;
    return over_tokens<T>(a, (a.rows + Work::kRows - 1) / Work::kRows, Work::kTokens, Work::kThreads, [&](const MatmulI8 &part) {
        const TileGrid grid = tile_grid(part, Work::kRows, Work::kTokens);
        CML_COUNT_LAUNCH("i8.matmul.staged");
        hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(grid.n_row_blocks * grid.n_token_blocks)), dim3(Work::kThreads), Work::kLds, st, part, grid);
    });
}

template <class T, bool STREAM>
static int launch_walk_stores(const MatmulI8 &a, hipStream_t st) {
    typedef TileWork<T, 2, 4, 4, 2, 2, false, true> Work;
    const auto kernel = matmul_i8_walk_kernel<T, 2, 4, 4, 2, STREAM>;
    static std::atomic<bool> raised{false};
    if (int rc = allow_lds(kernel, Work::kLds, raised)) return rc;
    CML_COUNT_LAUNCH("i8.matmul.walk");
    hipLaunchKernelGGL(kernel, dim3(256), dim3(Work::kThreads), Work::kLds, st, a, tile_grid(a, Work::kRows, Work::kTokens));
    CML_HIP_TRY(hipGetLastError());
    return CML_OK;
}
template <class T>
static int launch_walk(const MatmulI8 &a, hipStream_t st) {
    // An output of 96 MB and more, in whole lines, leaves past the caches, which do not hold it for the next kernel anyway (4096 tokens on 14336 x 4096, bf16, 117 MB: 242 us plain, 219
    // so, with a copy of it behind 284 and 280).  For smaller ones the next kernel pays (1024 tokens on 4096 x 4096: 24.0 and 21.6, with the copy 27.3 and 27.9), for rows that start
    // inside a line this one does (3461 tokens on 59669 x 128: 152 and 232).
    constexpr int kSize = sizeof(typename T::Bits);
    const bool lines = ((reinterpret_cast<uintptr_t>(a.out) | static_cast<uintptr_t>(a.out_stride * kSize)) & 127u) == 0;
    return lines && static_cast<int64_t>(a.n_tokens) * a.rows * kSize >= 96ll << 20 ? launch_walk_stores<T, true>(a, st) : launch_walk_stores<T, false>(a, st);
}

// What a call takes by tile, in microseconds: a start, then per workgroup that a compute unit runs `work` for each step of 128 values and `ends` for the tile;
// no tile is through its steps faster than `step` each, alone on its unit.  Fitted to one weight over and over, 1 - 4096 tokens on 64 x 512 to 128256 x 2048, so that smaller ones were in the
// caches; it has no term for memory.  With weights from memory (twelve shapes from 1024 x 4096 to 151936 x 1024, as many of each in turn as make 1.2 GB, 1 - 512 tokens) a call takes
// 1.1 to 2.4 times what it says, and yet the order of the tiles holds: the one that is picked takes 1.4 % more than the best one in the mean, 15 % at most (16 tokens on 14336 x 4096: 16.7 us, in
// tiles of 64 x 64 that ask for the weight past the caches 14.6); with small weights in the caches 1.8 % and 25 % (the same call: 14.8, in tiles of 64 x 32 11.9).
struct TileCost {
    int rows, tokens, per_unit;
    float start, step, work, ends;
};
constexpr TileCost kWalk{256, 256, 1, 3.0f, 1.12f, 0.85f, 6.2f},
    kTiles[] = {{256, 128, 1, 3.0f, 0.73f, 0.63f, 3.2f},   {128, 128, 1, 3.0f, 0.51f, 0.435f, 2.9f},   {64, 128, 2, 3.0f, 0.36f, 0.32f, 0.92f},
                {64, 64, 2, 3.0f, 0.236f, 0.213f, 0.5f},   {64, 32, 3, 3.0f, 0.213f, 0.174f, 0.4f},    {16, 16, 3, 2.5f, 0.054f, 0.049f, 0.425f},
                {32, 16, 2, 2.5f, 0.078f, 0.073f, 0.663f}, {16, 32, 3, 2.5f, 0.08f, 0.074f, 0.427f},   {32, 32, 2, 2.5f, 0.117f, 0.104f, 0.662f},
                {16, 64, 2, 2.5f, 0.136f, 0.124f, 0.755f}, {32, 64, 1, 2.5f, 0.052f, 0.153f, 2.217f}};
// The same for rows that start anywhere: two staged tiles, three slim ones.  Fitted to 1 - 3300 tokens on sixteen weight shapes: 0.3 % more than the best in the mean, 39 % at most.
constexpr TileCost kAnyTiles[] = {{128, 128, 1, 3.0f, 0.56f, 0.987f, 2.262f}, {64, 64, 2, 3.0f, 0.51f, 0.464f, 0.117f}, {16, 16, 3, 2.5f, 0.033f, 0.105f, 0.348f},
                                  {32, 16, 2, 2.5f, 0.063f, 0.168f, 0.506f},  {32, 32, 1, 2.5f, 0.163f, 0.227f, 0.764f}};
static float tile_cost(const MatmulI8 &a, const TileCost &c) {
    const int64_t tiles = static_cast<int64_t>((a.rows + c.rows - 1) / c.rows) * ((a.n_tokens + c.tokens - 1) / c.tokens);
    const float steps = static_cast<float>((a.cols + 127) / 128), one = c.work * steps + c.ends;
    if (&c == &kWalk) return c.start + std::max(c.step * steps, std::max(1.0f, 0.5f * static_cast<float>((tiles + 127) / 128)) * one);  // (half rounds)
    const int64_t full = tiles / (256 * c.per_unit), left = tiles - full * 256 * c.per_unit;
    return c.start + static_cast<float>(full * c.per_unit) * one + (left ? std::max(c.step * steps, static_cast<float>((left + 255) / 256) * one) : 0.0f);
}

// Variants: 0 the walk, 1 - 5 the first of kTiles, 6 / 7 tiles of 128 x 64 / 64 x 64 that ask for the weight past the caches, 8 - 13 the slim ones; 14 - 18 kAnyTiles.
template <int N>
static int cheapest(const MatmulI8 &a, const TileCost (&tiles)[N], float &least) {
    int best = 0;
    least = tile_cost(a, tiles[0]);
    for (int i = 1; i < N; i++) {
        const float c = tile_cost(a, tiles[i]);
        if (c < least) {
            least = c;
            best = i;
        }
    }
    return best;
}
static int choose_aligned(const MatmulI8 &a) {
    const int64_t bytes = static_cast<int64_t>(a.rows) * a.cols;
    // A weight of 96 MB and more is used once in a pass over a model: past the caches (128256 x 2048, 1 / 16 / 37 tokens: 52 / 55 / 59 us plain, 45 / 46 / 49 so), in the
    // tile that has two workgroups for every compute unit (32000 x 4096, 1 / 32 tokens: 128 x 64 31 / 29, 64 x 64 29 / 28; 48 tokens: 30 / 30, plain 24), where that is a tile for every unit
    // (4096 x 28672, one token: 62, plain and slim 25).  With weights from memory, 1 and 64 tokens, 128 x 64 / 64 x 64 past the caches: 65536 x 2048 23.4 and 26.0 / 26.6 and 32.0 us,
    // 151936 x 1024 32.7 and 39.8 / 33.3 and 43.7, 128256 x 2048 43.4 and 53.6 / 45.6 and 61.8; on 100352 x 4096 the smaller one is ahead, 81.4 and 93.2 / 74.2 and 91.1.
    if (bytes >= 96ll << 20 && a.n_tokens <= 64) {
        if ((a.rows + 127) / 128 >= 512) return 6;
        if (a.n_tokens <= 32 && (a.rows + 63) / 64 >= 256) return 7;
    }
    float least;
    const int best = cheapest(a, kTiles, least);
    if (a.rows >= 256 && a.n_tokens >= 256 && tile_cost(a, kWalk) < least) return 0;
    return best < 5 ? best + 1 : best + 3;
}
// Rows that start anywhere.
static int choose_any(const MatmulI8 &a) {
    float least;
    return 14 + cheapest(a, kAnyTiles, least);
}

template <class T>
static int launch_variant(int v, const MatmulI8 &a, hipStream_t st) {
    switch (v) {
        case 0: return launch_walk<T>(a, st);
        case 1: return launch_tile<T, 4, 2, 2, 2, 3, 1>(a, st);
        case 2: return launch_tile<T, 2, 2, 2, 2, 4, 1>(a, st);
        case 3: return launch_tile<T, 2, 4, 1, 1, 3, 2>(a, st);
        case 4: return launch_tile<T, 2, 2, 1, 1, 4, 2>(a, st);
        case 5: return launch_tile<T, 2, 1, 1, 1, 4, 3>(a, st);
        case 6: return launch_tile<T, 4, 1, 1, 2, 3, 2, true>(a, st);
        case 7: return launch_tile<T, 2, 2, 1, 1, 4, 2, true>(a, st);
        case 8: return launch_slim<T, 1, 1, 4, 3, false>(a, st);
        case 9: return launch_slim<T, 2, 1, 4, 3, false>(a, st);
        case 10: return launch_slim<T, 1, 2, 4, 2, false>(a, st);
        case 11: return launch_slim<T, 2, 2, 4, 2, false>(a, st);
        case 12: return launch_slim<T, 1, 4, 4, 2, false>(a, st);
        case 13: return launch_slim<T, 2, 4, 4, 2, false>(a, st);
        case 14: return launch_staged<T, 2>(a, st);
        case 15: return launch_staged<T, 1>(a, st);
        case 16: return launch_slim<T, 1, 1, 4, 1, true>(a, st);
        case 17: return launch_slim<T, 2, 1, 4, 1, true>(a, st);
        default: return launch_slim<T, 2, 2, 4, 1, true>(a, st);
    }
}

int launch_matmul_i8(const int8_t *q, int64_t q_stride, const float *scales, int64_t n_tokens, const int8_t *w, int64_t w_stride, const float *w_scales, int64_t rows, int64_t cols,
                     const float *bias, int dtype, void *out, int64_t out_stride, hipStream_t st) {
    // (the stride of a single row says nothing: whatever a caller has there, the row's address decides)
    if (n_tokens == 1) q_stride = 0;
    if (rows == 1) w_stride = 0;
    const MatmulI8 a{q, w, scales, w_scales, bias, out, q_stride, w_stride, out_stride, static_cast<int>(n_tokens), static_cast<int>(rows), static_cast<int>(cols)};
    const bool aligned = ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(w) | static_cast<uintptr_t>(q_stride | w_stride)) & 15u) == 0 &&
                         q_stride < (1 << 23) && w_stride < (1 << 23);  // (256 rows within 32 bits)
    const int forced = env_int("CAMELID_HIP_I8_TILE", 0) - 1;  // a variant, where it serves the call
    const bool near = q_stride < (1 << 26) && w_stride < (1 << 26);  // (64 rows within 32 bits)
    int v = aligned ? choose_aligned(a) : near ? choose_any(a) : 15;
    if (near && forced >= (aligned ? 0 : 14) && forced <= 18 && !(forced == 0 && (rows < 256 || n_tokens < 256))) v = forced;
    return with_type(dtype, [&](auto t) { return launch_variant<decltype(t)>(v, a, st); });
}

}  // namespace cml
