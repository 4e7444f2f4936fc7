// The selective scan of token sequences, what its kernels share.  u, delta, z (batch, token, channel), B and C (batch, token, group, state); per channel a
// state h of N values,
//     step = softplus(delta + bias),   h_t = exp(step_t A) h_(t-1) + step_t u_t B_t,   y_t = (C_t . h_t + D u_t) silu(z_t).
// Channels are neighbours in memory, tokens are rows (the framework's scan of maps, selective_scan.hip, has positions for neighbours): a wavefront takes kCh = 16, 32 or 64
// channels and walks the tokens one by one in tiles of 16.  A channel's states lie with kSets = 4, 2 or 1 lanes, 4 kM with each:
//     lane = channel % 4 + 4 (set + kSets (channel / 4)),   state n = 4 kSets m + 4 set + v of accumulator v = 0 .. 3 of m < kM,
// which is how v_mfma_f32_4x4x1 leaves 16 products of 4 states and 4 channels: h = mfma(B, step u, a h) adds the outer product of B_t and step u in one
// instruction beside the vector ones, fp32 and fused, where a product and a fused addition for each value were a third of them.
//
// Sequences.  Rows of a batch, or packed one behind another in a batch of one (cu: their places); a tile never holds tokens of two.  The token axis is
// cut into segments that run side by side where channels are too few for the chip.
#pragma once
#include "scan_common.h"

namespace ss2d {

constexpr int kTsTile = 16;          // tokens of a tile
constexpr int kTsGrid = 64;          // tokens of a segment at least
constexpr int kTsMaxState = 64;
constexpr int64_t kTsLaunch = 0xffffffff;                            // threads of a launch

struct TsArgs {
    const void *u, *delta, *B, *C, *z;
    const float *A, *D, *bias, *initial;
    const int32_t *cu;
    void *out;
    float *final, *kept;             // kept: [batch][token / keep][channel][state], the state before every keep-th token
    int64_t u_b, u_t, dl_b, dl_t, z_b, z_t, B_b, B_t, B_g, C_b, C_t, C_g;
    int32_t batch, tokens, dim, N, groups, per_group, n_seqs, softplus;
    int32_t near;                    // offsets inside a tile fit 32 bits
    int32_t wgs;                     // workgroups (of four wavefronts' channels) to a group
    int32_t seg_len, n_segs, keep, n_kept;                           // n_kept: kept states of a row
    // workspace: of every segment but the last [batch][segment][channel](..)
    float *end, *sums;               // state behind it (N), from zeros or its last sequence's start; its steps' sum
    float *enter;                    // state before segment + 1 (N)
    int32_t *flags;                  // [batch][segment]: TsCarry
};

// Tokens of n segments, a multiple of `keep`: a segment begins with a kept state
inline int ts_seg_len(int64_t tokens, int64_t n, int keep) {
    n = n < 1 ? 1 : n;
    int64_t len = ((tokens + n - 1) / n + keep - 1) / keep * keep;
    len = len < kTsGrid ? kTsGrid : len;
    return (int)len;
}
inline int ts_sets(int N) { return N <= 4 ? 1 : N <= 8 ? 2 : 4; }
// Whole wavefronts of channels, states that fill their lanes, offsets inside a tile that fit 32 bits: the kernels without masks
inline bool ts_quick(const TsArgs &a) { return a.near && a.per_group % (kWave / ts_sets(a.N)) == 0 && (a.N == 4 || a.N == 8 || a.N == 16 || a.N == 32 || a.N == 64); }
// Tokens between the states that the forward keeps for the gradients: 4 bytes per token and channel where the states fill their lanes.  (Of 16 states, every 64th token
// takes a quarter of the memory and the gradients a second walk over every piece: their kernel, before wavefronts kept together, 310 us where it was 278, 4 x 2048 tokens of 2048
// channels.)
inline int ts_keep(int N) { return N <= 16 ? 16 : N <= 32 ? 32 : 64; }

// The gradients' sums have a thread to a value of B, and one to a value of A, D and the bias: launches count them in 32 bits
inline bool ts_sums_fit(const TsArgs &a) {
    constexpr int64_t kMost = kTsLaunch / kBlock * kBlock;
    const __int128 values = (__int128)a.batch * a.tokens * a.groups * a.N;
    return values <= kMost && (int64_t)a.dim * (a.N + 2) <= kMost;
}

enum TsCarry { kTsNothing, kTsStarts, kTsThrough };                  // what a segment hands on: nothing, its last sequence began in it, it lies inside one

// Wavefronts of a workgroup of the gradients' kernel: their states in LDS are 4 kM^2 KB each
template <int kM> constexpr int kTsBwdWaves = kM == 4 ? 2 : 4;

// The gradients' further arguments
struct TsBwdArgs {
    TsArgs f;
    const void *dout;
    const float *dfinal;
    void *du, *ddelta, *dz;
    float *dinitial;
    int64_t do_b, do_t;
    // what is handed from behind is found from shorter segments, `each` of them to one of the gradients': of the `slots` of them behind the first `each`, as end, sums, enter
    // and flags, the other way
    float *left, *gsums, *behind;
    int32_t *gflags;
    int32_t each, slots, left_wgs;   // left_wgs: their workgroups to a group
    float *pBC;                      // [workgroup of a group][batch][token][group][state][B, C]: sums over a workgroup's channels
    float *pA;                       // [batch][segment][channel][state]
    float *pD;                       // [batch][segment][D, bias][channel]
};

struct TsSpan { int32_t seq, lo, hi; };                              // a sequence and its tokens; seq -1: tokens of none

// The sequence of token t (uniform).  Whatever cu holds, lo <= t < hi, all inside 0 .. tokens.
__device__ __forceinline__ TsSpan ts_span_at(const int32_t *__restrict__ cu, int n_seqs, int tokens, int b, int t) {
    if (!cu) return {b, 0, tokens};
    auto place = [&](int i) { return min(max(cu[i], 0), tokens); };
    const int first = place(0), last = place(n_seqs);
    if (t < first) return {-1, 0, first};
    if (last <= t) return {-1, last, tokens};
    int l = 0, r = n_seqs, lo = first, hi = last;
    while (r - l > 1) {
        const int m = l + ((r - l) >> 1), at = place(m);
        if (at <= t) { l = m; lo = at; }
        else { r = m; hi = at; }
    }
    return {l, lo, hi};
}

// ---- four neighbouring values, n of them there, at any address of their type ------------------------------------------------------
template <typename T> struct Raw4 { uint32_t w[sizeof(T)]; };

template <typename T> __device__ __forceinline__ Raw4<T> ts_load4(const T *p, int n, bool whole) {
    Raw4<T> r;
    if (whole) {                                                     // (uniform: every lane has its four)
        typedef uint32_t here __attribute__((ext_vector_type(sizeof(T)), aligned(sizeof(T))));
        const here v = *reinterpret_cast<const here *>(p);
#pragma unroll
        for (int i = 0; i < (int)sizeof(T); ++i) r.w[i] = v[i];
        return r;
    }
#pragma unroll
    for (int i = 0; i < (int)sizeof(T); ++i) r.w[i] = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (i >= n) break;
        if constexpr (sizeof(T) == 4) r.w[i] = f32_to_bits(p[i]);
        else r.w[i / 2] |= (uint32_t)p[i].bits << (i & 1) * 16;
    }
    return r;
}
// ... at a uniform place and 32 bits' worth of bytes on
template <typename T> __device__ __forceinline__ Raw4<T> ts_load4_at(const T *base, uint32_t bytes) {
    return ts_load4<T>(reinterpret_cast<const T *>(reinterpret_cast<const char *>(base) + bytes), 4, true);
}
template <typename T> __device__ __forceinline__ void ts_widen(const Raw4<T> &r, float (&v)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 4) v[i] = bits_to_f32(r.w[i]);
        else v[i] = i & 1 ? unpack_hi<T>(r.w[i / 2]) : unpack_lo<T>(r.w[i / 2]);
    }
}
// kStreamed: past the caches, for results that the launch does not read again.  The gradients gain 2 % by it, the forward, which waits for no memory, loses 1 %.
template <typename T, bool kStreamed = false> __device__ __forceinline__ void ts_store4(T *p, int n, bool whole, const float (&v)[4]) {
    if (whole) {
        typedef uint32_t here __attribute__((ext_vector_type(sizeof(T)), aligned(sizeof(T))));
        here w;
        if constexpr (sizeof(T) == 4) w = here{f32_to_bits(v[0]), f32_to_bits(v[1]), f32_to_bits(v[2]), f32_to_bits(v[3])};
        else w = here{pack2_from_f32<T>(v[0], v[1]), pack2_from_f32<T>(v[2], v[3])};
        if constexpr (kStreamed) __builtin_nontemporal_store(w, reinterpret_cast<here *>(p));
        else *reinterpret_cast<here *>(p) = w;
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (i < n) p[i] = from_f32<T>(v[i]);
}

// ---- lanes -----------------------------------------------------------------------------------------------------------------------
// What a lane does: a channel's states where it computes, a token's four channels where tiles come in and go out.
template <int kSets, int kM> struct TsLane {
    static constexpr int kCh = kWave / kSets, kStates = 4 * kSets * kM;
    static constexpr int kCols = kCh / 4, kRows = kWave / kCols, kRounds = kTsTile / kRows;      // of a tile: lanes to a token, tokens to a round
    static constexpr int kPieces = kSets * kM, kBcRows = kWave / kPieces;                        // of a row of B or C: four states to a lane; tokens to a round
    static constexpr int kBcRounds = kBcRows >= kTsTile ? 1 : kTsTile / kBcRows;
    static constexpr int kPairPitch = 2 * kCh + 4, kPitch = kCh + 4;
    int lane, chan, set, col;                                        // computing
    int row, at;                                                     // staging: token of a round, first of its four channels
    int piece, bc_row;                                               // B and C
    __device__ __forceinline__ explicit TsLane(int lane_) : lane(lane_) {
        col = lane & 3; set = (lane >> 2) % kSets; chan = 4 * (lane / (4 * kSets)) + col;
        row = lane / kCols; at = lane % kCols * 4;
        piece = lane % kPieces; bc_row = lane / kPieces;
    }
    __device__ __forceinline__ int state(int m) const { return 4 * kSets * m + 4 * set; }        // the first of its four
};

__device__ __forceinline__ floatx4_t ts_outer(float row, float col, floatx4_t c) { return __builtin_amdgcn_mfma_f32_4x4x1f32(row, col, c, 0, 0, 0); }

// Values of a lane that stand for no state of a channel: cleared behind what the matrix instruction makes of them, 0 times a step u or a step that may be infinite
template <int kSets, int kM> __device__ __forceinline__ void ts_clear_others(floatx4_t &v, int m, int N, const TsLane<kSets, kM> &l, bool there) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = there && l.state(m) + i < N ? v[i] : 0.0f;
}

// A channel's states of a lane from and to [channel][state] memory
template <int kSets, int kM> __device__ __forceinline__ void ts_read_state(const float *from, int N, const TsLane<kSets, kM> &l, bool there, floatx4_t (&h)[kM]) {
    typedef float here __attribute__((ext_vector_type(4), aligned(4)));
#pragma unroll
    for (int m = 0; m < kM; ++m) {
        const int n = l.state(m);
        h[m] = floatx4_t{0, 0, 0, 0};
        if (!there || !from) continue;
        if (n + 4 <= N) h[m] = *reinterpret_cast<const here *>(from + n);
        else
#pragma unroll
            for (int v = 0; v < 3; ++v)
                if (n + v < N) h[m][v] = from[n + v];
    }
}
template <int kSets, int kM> __device__ __forceinline__ void ts_write_state(float *to, int N, const TsLane<kSets, kM> &l, bool there, const floatx4_t (&h)[kM]) {
    typedef float here __attribute__((ext_vector_type(4), aligned(4)));
    if (!there) return;
#pragma unroll
    for (int m = 0; m < kM; ++m) {
        const int n = l.state(m);
        if (n + 4 <= N) *reinterpret_cast<here *>(to + n) = h[m];
        else
#pragma unroll
            for (int v = 0; v < 3; ++v)
                if (n + v < N) to[n + v] = h[m][v];
    }
}

// v[t] of a tile's 16 tokens summed over a channel's sets: 16 / kSets tokens from kSets' share on are left with each, in v[0 ..].
template <int kSets> __device__ __forceinline__ void ts_sum_sets(float (&v)[16]) {
    if constexpr (kSets == 4) sum_over_quads(v);
    if constexpr (kSets == 2) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {                                // lanes of set 0 take the first eight from the lanes four above, of set 1 the others from below
            const float low = v[i] + dpp_move<0x104>(0.0f, v[i]), high = v[8 + i] + dpp_move<0x114>(0.0f, v[8 + i]);
            v[i] = threadIdx.x & 4 ? high : low;
        }
    }
}

// Wavefronts of a SIMD that walk as far keep together: the oldest would run ahead and leave the last ones a SIMD that they cannot fill.  The nearer the end,
// the lower the priority: in the first half, to three quarters, seven eighths, behind.  32768 tokens 476 -> 418 us, 4 x 2048 with their gradients 447 -> 415 (when 32768 tokens took 430, bounds nearer the
// end, 15/16, 31/32 and 63/64, 467, quarters 447, a turn of four priorities every four tiles 437).  Beside other work: a scan of 8192 tokens and kernels of another stream end together as soon as
// without priorities or sooner (0 to 7 %), the others being served later: products of 2048^3 42 us in place of 37 (27 alone), copies of 256 MB 151 and 146 (100), GELUs of 8 MB 9.9 and 9.2 (6).
__device__ __forceinline__ void ts_keep_together(int left, int of) {
    if (2 * left > of) __builtin_amdgcn_s_setprio(3);
    else if (4 * left > of) __builtin_amdgcn_s_setprio(2);
    else if (8 * left > of) __builtin_amdgcn_s_setprio(1);
    else __builtin_amdgcn_s_setprio(0);
}

// What a segment hands on of what comes into it, with its own: by its decays' product, exp2(2 A2_half sum), in two halves, so that neither leaves the range of fp32 before the state
// would.  An infinite state stays what it is by decays that are numbers, however small their product; a decay of 0 (of an infinite step or A) makes NaN of it.
__device__ __forceinline__ float ts_handed_on(float carry, float A2_half, float sum, float own) {
    const float of_two = A2_half * sum, half = __builtin_amdgcn_exp2f(of_two);
    if (fabsf(carry) == __builtin_inff()) return (fabsf(of_two) < __builtin_inff() ? carry : carry * half) + own;
    return fmaf(carry * half, half, own);
}

__device__ __forceinline__ float ts_sigmoid(float x) { return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-kLog2e * x)); }

}  // namespace ss2d
