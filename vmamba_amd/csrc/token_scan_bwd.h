// Gradients of the selective scan of token sequences (token_scan.h).  With dy_t = dout_t silu(z_t) and a_t = exp(step_t A), the other recurrence goes
// from the last token to the first,
//     g_t = dy_t C_t + a_(t+1) g_(t+1),
// and of it and the states come   dC_t = sum over channels dy_t h_t,   dB_t = sum over channels step_t u_t g_t,   with s_t = g_t . B_t and
// w_t = a_t g_t h_(t-1):   du_t = D dy_t + step_t s_t,   dstep_t = u_t s_t + w_t . A,   dA = sum over t of step_t w_t,   dD = sum dy_t u_t.
//
// The states are found again from those that the forward kept (ts_keep): of a piece of the tokens from one to the next, inside one sequence, the states
// before every 8th are left in LDS, then it is walked backwards by eights, whose states and decays stay in registers.  Segments of the token axis run side by side;
// what a later one hands to an earlier one is found first, from its own tokens (ts_left_kernel), and joined.  Sums over channels: a wavefront's by lane moves, two tokens'
// dB and dC of a lane's four states at once, a workgroup's four through LDS, all workgroups' from memory in a fixed order.  No atomics.
//
// Vector instructions bound it, 1603 a tile of 4096 values of states: 800 for states, decays and products, 256 for sums over channels, 70 over states; they are issued in 81 % of the
// CUs' busy cycles, of two wavefronts to a SIMD, all that 230 registers leave (three spill: 613 us in place of 414 of the whole case).  4 x 2048 tokens of 2048 channels, 16 states,
// bf16: 242 us, what later segments hand back 38, joins and sums 25, and the forward with kept states 109.
#pragma once
#include "token_scan.h"

namespace ss2d {

constexpr int kTsSub = 8;                                            // tokens between two states in LDS

// v[8 token + 4 is_C + state] of 16 summed over a wavefront's channels; entry 8 (lane bit 5) + 4 (bit 4) + 2 (bit 1) + (bit 0) is left with each lane.
template <int kSets> __device__ __forceinline__ float ts_sum_channels(float (&v)[16], int lane) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const auto r = __builtin_amdgcn_permlane32_swap(f32_to_bits(v[i]), f32_to_bits(v[i + 8]), false, false);
        v[i] = bits_to_f32(r[0]) + bits_to_f32(r[1]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const auto r = __builtin_amdgcn_permlane16_swap(f32_to_bits(v[i]), f32_to_bits(v[i + 4]), false, false);
        v[i] = bits_to_f32(r[0]) + bits_to_f32(r[1]);
        if constexpr (kSets < 4) v[i] += dpp_move<0x128>(0.0f, v[i]);          // row_ror:8
        if constexpr (kSets < 2) v[i] += dpp_move<0x124>(0.0f, v[i]);          // row_ror:4
    }
    auto halves = [&](float a, float b, bool upper, auto move) { return (upper ? b : a) + move(upper ? a : b); };
    auto by1 = [](float x) { return dpp_move<0xB1>(0.0f, x); };
    auto by2 = [](float x) { return dpp_move<0x4E>(0.0f, x); };
    const bool odd = lane & 1, high = lane & 2;
    return halves(halves(v[0], v[1], odd, by1), halves(v[2], v[3], odd, by1), high, by2);
}

// What a segment hands to the one before it, from its own tokens: a_t g_t of its first token
template <typename T, int kSets, int kM, bool kQuick>
__global__ __launch_bounds__(kBlock, 3) void ts_left_kernel(const TsBwdArgs q) {
    using L = TsLane<kSets, kM>;
    const TsArgs &p = q.f;
    __shared__ __align__(16) float s_all[kWavesPerWg][kTsTile * (L::kPairPitch + L::kStates)];
    const L l(threadIdx.x & (kWave - 1));
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    float *s_step = s_all[wave], *s_C = s_step + kTsTile * L::kPairPitch;
    uint32_t id = xcd_contiguous_id(blockIdx.x, gridDim.x);
    const int wg = (int)(id % (uint32_t)p.wgs); id /= (uint32_t)p.wgs;
    const int g = (int)(id % (uint32_t)p.groups); id /= (uint32_t)p.groups;
    const int segs = q.slots, seg = (int)(id % (uint32_t)segs) + q.each, b = (int)(id / (uint32_t)segs);
    const int first = (wg * kWavesPerWg + wave) * L::kCh, n_chan = min(L::kCh, p.per_group - first);
    if (n_chan <= 0) return;
    const int c0 = g * p.per_group + first, s0 = seg * p.seg_len, s1 = s0 + min(p.seg_len, p.tokens - s0);
    const bool whole = kQuick || n_chan == L::kCh, there = kQuick || l.chan < n_chan;
    const int mine = kQuick ? 4 : min(max(n_chan - l.at, 0), 4), at = mine > 0 ? l.at : 0, d = c0 + (kQuick ? l.chan : min(l.chan, n_chan - 1));
    const TsSpan sp = ts_span_at(p.cu, p.n_seqs, p.tokens, b, s0);
    const int carry = sp.seq < 0 || sp.lo >= s0 ? kTsNothing : sp.hi <= s1 ? kTsStarts : kTsThrough;
    const int64_t slot = (int64_t)b * segs + seg - q.each;
    if (wg == 0 && g == 0 && threadIdx.x == 0) q.gflags[slot] = carry;
    if (carry == kTsNothing) return;

    const T *dl = (const T *)p.delta + (int64_t)b * p.dl_b + c0, *dout = (const T *)q.dout + (int64_t)b * q.do_b + c0;
    const T *z = p.z ? (const T *)p.z + (int64_t)b * p.z_b + c0 : nullptr, *Cp = (const T *)p.C + (int64_t)b * p.C_b + (int64_t)g * p.C_g;
    const int N = kQuick ? L::kStates : p.N, bc_n = kQuick ? 4 : min(max(N - 4 * l.piece, 0), 4), bc_at = bc_n > 0 ? 4 * l.piece : 0;
    const bool bc_whole = kQuick || N == L::kStates;
    float bias[4], sum[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 4; ++i) bias[i] = p.bias && i < mine ? p.bias[c0 + at + i] : 0.0f;
    floatx4_t A2[kM], ga[kM];
    ts_read_state<kSets, kM>(p.A + (int64_t)d * N, N, l, true, A2);
    ts_read_state<kSets, kM>(carry == kTsStarts && q.dfinal ? q.dfinal + ((int64_t)sp.seq * p.dim + d) * N : nullptr, N, l, there, ga);
#pragma unroll
    for (int m = 0; m < kM; ++m) A2[m] *= kLog2e;
    Raw4<T> ro[L::kRounds], rd[L::kRounds], rz[L::kRounds], rC[L::kBcRounds];
    auto request = [&](int from, int to) {
        if constexpr (kQuick) {                                      // (a uniform base, and 32 bits from there on)
            auto row_of = [&](int k) { return (uint32_t)min(k, to - 1 - from); };
#pragma unroll
            for (int r = 0; r < L::kRounds; ++r) {
                const uint32_t k = row_of(r * L::kRows + l.row);
                ro[r] = ts_load4_at<T>(dout + from * q.do_t, (k * (uint32_t)q.do_t + (uint32_t)at) * (uint32_t)sizeof(T));
                rd[r] = ts_load4_at<T>(dl + from * p.dl_t, (k * (uint32_t)p.dl_t + (uint32_t)at) * (uint32_t)sizeof(T));
                if (z) rz[r] = ts_load4_at<T>(z + from * p.z_t, (k * (uint32_t)p.z_t + (uint32_t)at) * (uint32_t)sizeof(T));
            }
#pragma unroll
            for (int r = 0; r < L::kBcRounds; ++r)
                rC[r] = ts_load4_at<T>(Cp + from * p.C_t, (row_of(r * L::kBcRows + l.bc_row) * (uint32_t)p.C_t + (uint32_t)bc_at) * (uint32_t)sizeof(T));
            return;
        }
#pragma unroll
        for (int r = 0; r < L::kRounds; ++r) {
            const int64_t k = min(from + r * L::kRows + l.row, to - 1);
            ro[r] = ts_load4<T>(dout + at + k * q.do_t, mine, whole);
            rd[r] = ts_load4<T>(dl + at + k * p.dl_t, mine, whole);
            if (z) rz[r] = ts_load4<T>(z + at + k * p.z_t, mine, whole);
        }
#pragma unroll
        for (int r = 0; r < L::kBcRounds; ++r) rC[r] = ts_load4<T>(Cp + (int64_t)min(from + r * L::kBcRows + l.bc_row, to - 1) * p.C_t + bc_at, bc_n, bc_whole);
    };
    int e = min(sp.hi, s1), t = (e - 1) & ~(kTsTile - 1);            // (segments begin on multiples of a tile)
    request(t, e);
    for (;;) {
        const int n = e - t;
        ts_keep_together(e - s0, s1 - s0);
#pragma unroll
        for (int r = 0; r < L::kRounds; ++r) {
            const int k = r * L::kRows + l.row;
            float ov[4], dv[4], step[4];
            ts_widen<T>(ro[r], ov);
            ts_widen<T>(rd[r], dv);
            if (z) {
                float zv[4];
                ts_widen<T>(rz[r], zv);
#pragma unroll
                for (int i = 0; i < 4; ++i) ov[i] *= zv[i] * ts_sigmoid(zv[i]);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                step[i] = p.softplus ? softplus_log2(fmaf(dv[i], kLog2e, bias[i] * kLog2e)) : dv[i] + bias[i];
                const bool in = k < n && (whole || i < mine);
                step[i] = in ? step[i] : 0.0f;
                ov[i] = in ? ov[i] : 0.0f;
                sum[i] += step[i];
            }
            float *to = s_step + k * L::kPairPitch + 2 * l.at;
            *reinterpret_cast<float4 *>(to) = make_float4(step[0], ov[0], step[1], ov[1]);
            *reinterpret_cast<float4 *>(to + 4) = make_float4(step[2], ov[2], step[3], ov[3]);
        }
#pragma unroll
        for (int r = 0; r < L::kBcRounds; ++r) {
            const int k = r * L::kBcRows + l.bc_row;
            if (L::kBcRows > kTsTile && k >= kTsTile) continue;
            float v[4];
            ts_widen<T>(rC[r], v);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = k < n ? v[i] : 0.0f;
            *reinterpret_cast<float4 *>(s_C + k * L::kStates + 4 * l.piece) = bc_n > 0 ? make_float4(v[0], v[1], v[2], v[3]) : make_float4(0, 0, 0, 0);
        }
        const bool more = t > s0;
        if (more) request(t - kTsTile, t);
        __builtin_amdgcn_sched_barrier(0);
        wave_lds_sync();
        auto walk = [&](auto all) {                                  // all: the tile has its 16 tokens (those it has not are not walked, as in the forward)
#pragma unroll
            for (int k = kTsTile - 1; k >= 0; --k) {
                if (!decltype(all)::value && k >= n) continue;
                const float2 pair = *reinterpret_cast<const float2 *>(s_step + k * L::kPairPitch + 2 * l.chan);
#pragma unroll
                for (int m = 0; m < kM; ++m) {
                    const floatx4_t gr = ts_outer(s_C[k * L::kStates + l.state(m) + l.col], pair.y, ga[m]);
#pragma unroll
                    for (int v = 0; v < 4; ++v) ga[m][v] = __builtin_amdgcn_exp2f(pair.x * A2[m][v]) * gr[v];
                }
            }
        };
        if (n == kTsTile) walk(std::true_type{});
        else walk(std::false_type{});
        wave_lds_sync();
        if (!more) break;
        e = t;
        t -= kTsTile;
    }
    ts_write_state<kSets, kM>(q.left + (slot * p.dim + d) * N, N, l, there, ga);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int over = L::kCols; over < kWave; over *= 2) sum[i] += __shfl_xor(sum[i], over, kWave);
        if (l.row == 0 && i < mine) q.gsums[slot * p.dim + c0 + at + i] = sum[i];
    }
}

// What enters every segment but the last from behind (as ts_join_kernel, the other way)
static __global__ __launch_bounds__(kBlock) void ts_join_left_kernel(const TsBwdArgs q, uint32_t per_row) {
    const TsArgs &p = q.f;
    const uint32_t item = blockIdx.x * kBlock + threadIdx.x;
    const int b = (int)blockIdx.y, segs = q.slots;
    if (item >= per_row) return;
    const uint32_t d = item / (uint32_t)p.N;
    const float A2 = 0.5f * kLog2e * p.A[item];
    const float *left = q.left + (int64_t)b * segs * per_row + item, *sums = q.gsums + (int64_t)b * segs * p.dim + d;
    const int32_t *flags = q.gflags + (int64_t)b * segs;
    float *behind = q.behind + (int64_t)b * segs * per_row + item;
    constexpr int kFly = 8;
    float carry = 0.0f;
    for (int s0 = segs - 1; s0 >= 0; s0 -= kFly) {
        float own[kFly], sum[kFly];
        int flag[kFly];
#pragma unroll
        for (int i = 0; i < kFly; ++i) {
            const int s = max(s0 - i, 0);
            own[i] = left[(int64_t)s * per_row];
            sum[i] = sums[(int64_t)s * p.dim];
            flag[i] = flags[s];
        }
#pragma unroll
        for (int i = 0; i < kFly; ++i) {
            if (s0 - i < 0) break;
            if (flag[i] == kTsThrough && carry != 0.0f) {
                carry = ts_handed_on(carry, A2, sum[i], own[i]);
            } else {
                carry = flag[i] == kTsNothing ? 0.0f : own[i];
            }
            behind[(int64_t)(s0 - i) * per_row] = carry;
        }
    }
}

// Arguments that a piece needs once, read again each time: held in scalar registers with the others, which are more than there are, they would push those out
typedef const __attribute__((address_space(4))) TsBwdArgs *TsRare;
__device__ __forceinline__ TsRare ts_rare_args() {
    TsRare q = (TsRare)__builtin_amdgcn_kernarg_segment_ptr();       // (the kernel's one argument)
    asm volatile("" : "+s"(q));
    return q;
}

enum TsEnds { kTsWhole, kTsLast, kTsPacked };

struct TsPiece { TsSpan sp; int32_t a, e; };                         // tokens a .. e - 1 of one sequence (or of none), from a kept state or a sequence's start on

// kQuick: whole wavefronts of channels, states that fill their lanes, and offsets inside a tile that fit 32 bits.  kEnds: where pieces may begin and end
// inside eight tokens that are walked together: nowhere, at the last token, anywhere (packed sequences).  Tokens that a piece has not are not walked: their steps of 0 and their
// products with 0 would be NaN of an A, a state or a gradient that is infinite.
template <typename T, int kSets, int kM, bool kQuick, TsEnds kEnds>
__global__ __launch_bounds__(kWave * kTsBwdWaves<kM>, kM > 1 || kSets == 1 ? 1 : 2) void ts_grad_kernel(const TsBwdArgs q) {
    using L = TsLane<kSets, kM>;
    const TsArgs &p = q.f;
    constexpr bool kPacked = kEnds == kTsPacked, kRagged = kEnds != kTsWhole;
    constexpr int kWaves = kTsBwdWaves<kM>, kThreads = kWave * kWaves, kRow = 4 * L::kCh + 4, kQuarter = 4 * kSets;
    constexpr int kKeep = kTsTile * kM, kSlots = kKeep / kTsSub;     // (ts_keep); states in LDS of a piece
    constexpr int kSlot = 4 * kWave * kM;                            // floats of a state in LDS, [m][lane][4]; later the sums of its eight tokens, [m][token][state][B, C]
    constexpr int kTurns = kM == 1 ? 2 : 1;                          // pieces take turns in them, so that one barrier to a piece is enough
    // of a tile: step, step u (later s), dy and u of every channel; B; C; w . A and y of every channel
    __shared__ __align__(16) float s_tok_all[kWaves][kTsTile * (kRow + 2 * L::kStates + 2 * L::kPitch)];
    __shared__ __align__(16) float s_slot_all[kTurns][kWaves][kSlots * kSlot];
    const L l(threadIdx.x & (kWave - 1));
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    float *s_tok = s_tok_all[wave], *s_B = s_tok + kTsTile * kRow, *s_C = s_B + kTsTile * L::kStates, *s_q = s_C + kTsTile * L::kStates, *s_y = s_q + kTsTile * L::kPitch;
    uint32_t id = xcd_contiguous_id(blockIdx.x, gridDim.x);
    const int wg = (int)(id % (uint32_t)p.wgs); id /= (uint32_t)p.wgs;
    const int g = (int)(id % (uint32_t)p.groups); id /= (uint32_t)p.groups;
    const int seg = (int)(id % (uint32_t)p.n_segs), b = (int)(id / (uint32_t)p.n_segs);
    const int first = (wg * kWaves + wave) * L::kCh, n_chan = min(L::kCh, p.per_group - first);
    const bool works = n_chan > 0;                                   // (a wavefront without channels meets the others' barriers)
    const int n_works = min(kWaves, (p.per_group - wg * kWaves * L::kCh + L::kCh - 1) / L::kCh);
    const int c0 = g * p.per_group + (works ? first : 0), s0 = seg * p.seg_len, s1 = s0 + min(p.seg_len, p.tokens - s0);
    const bool whole = kQuick || n_chan == L::kCh, there = kQuick || l.chan < n_chan;
    const int mine = kQuick ? 4 : min(max(n_chan - l.at, 0), 4), at = mine > 0 ? l.at : 0, d = c0 + (kQuick ? l.chan : max(min(l.chan, n_chan - 1), 0));
    const T *u = (const T *)p.u + (int64_t)b * p.u_b + c0, *dl = (const T *)p.delta + (int64_t)b * p.dl_b + c0;
    const T *dout = (const T *)q.dout + (int64_t)b * q.do_b + c0, *z = p.z ? (const T *)p.z + (int64_t)b * p.z_b + c0 : nullptr;
    const T *Bp = (const T *)p.B + (int64_t)b * p.B_b + (int64_t)g * p.B_g, *Cp = (const T *)p.C + (int64_t)b * p.C_b + (int64_t)g * p.C_g;
    const int64_t row0 = (int64_t)b * p.tokens * p.dim + c0;
    T *du = (T *)q.du + row0, *dd = (T *)q.ddelta + row0, *dz = (T *)q.dz + row0;
    const int N = kQuick ? L::kStates : p.N, bc_n = kQuick ? 4 : min(max(N - 4 * l.piece, 0), 4), bc_at = bc_n > 0 ? 4 * l.piece : 0;
    const bool bc_whole = kQuick || N == L::kStates;
    float bias[4], skip[4], sum_D[4] = {0, 0, 0, 0}, sum_bias[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        bias[i] = p.bias && i < mine ? p.bias[c0 + at + i] : 0.0f;
        skip[i] = p.D && i < mine ? p.D[c0 + at + i] : 0.0f;
    }
    floatx4_t A2[kM], ga[kM], dA[kM], next_h[kM];
    ts_read_state<kSets, kM>(p.A + (int64_t)d * N, N, l, works && there, A2);
    // values of a lane that stand for no state, or for none of the group's channels: 0 behind every matrix instruction, which may make NaN of them
    auto cleared = [&](floatx4_t v, int m) {
        if constexpr (!kQuick) ts_clear_others<kSets, kM>(v, m, N, l, there);
        return v;
    };
#pragma unroll
    for (int m = 0; m < kM; ++m) {
        A2[m] *= kLog2e;
        if (!kQuick)
#pragma unroll
            for (int v = 0; v < 4; ++v) A2[m][v] = l.state(m) + v < N ? A2[m][v] : -1.0f;            // (a decay that is a number even of an infinite step)
        ga[m] = dA[m] = floatx4_t{0, 0, 0, 0};
    }
    auto of_seq = [&](const float *states, int seq) { return states ? states + ((int64_t)seq * p.dim + d) * N : nullptr; };
    if (kPacked && ts_rare_args()->dinitial && works)                                 // sequences without tokens, dealt out over the segments
        for (uint32_t i = seg; i < (uint32_t)p.n_seqs; i += p.n_segs) {
            const int lo = min(max(p.cu[i], 0), p.tokens), hi = min(max(p.cu[i + 1], 0), p.tokens);
            if (hi > lo) continue;
            floatx4_t h[kM];
            ts_read_state<kSets, kM>(of_seq(ts_rare_args()->dfinal, (int)i), N, l, there, h);
            ts_write_state<kSets, kM>(ts_rare_args()->dinitial + ((int64_t)i * p.dim + d) * N, N, l, there, h);
        }

    Raw4<T> ru[L::kRounds], rd[L::kRounds], rz[L::kRounds], ro[L::kRounds], rB[L::kBcRounds], rC[L::kBcRounds];
    // tokens of the tile from `base` on, those inside a .. e - 1; the first walk needs no gradients
    auto request = [&](int base, int a, int e, bool second) {
        if constexpr (kQuick) {                                      // (a uniform base, and 32 bits from there on)
            auto row_of = [&](int k) { return (uint32_t)max(min(k, e - 1 - base), a - base); };
#pragma unroll
            for (int r = 0; r < L::kRounds; ++r) {
                const uint32_t k = row_of(r * L::kRows + l.row);
                ru[r] = ts_load4_at<T>(u + (int64_t)base * (int32_t)p.u_t, (k * (uint32_t)(int32_t)p.u_t + (uint32_t)at) * (uint32_t)sizeof(T));
                rd[r] = ts_load4_at<T>(dl + (int64_t)base * (int32_t)p.dl_t, (k * (uint32_t)(int32_t)p.dl_t + (uint32_t)at) * (uint32_t)sizeof(T));
                if (second) {
                    ro[r] = ts_load4_at<T>(dout + (int64_t)base * (int32_t)q.do_t, (k * (uint32_t)(int32_t)q.do_t + (uint32_t)at) * (uint32_t)sizeof(T));
                    if (z) rz[r] = ts_load4_at<T>(z + (int64_t)base * (int32_t)p.z_t, (k * (uint32_t)(int32_t)p.z_t + (uint32_t)at) * (uint32_t)sizeof(T));
                }
            }
#pragma unroll
            for (int r = 0; r < L::kBcRounds; ++r) {
                const uint32_t k = row_of(r * L::kBcRows + l.bc_row);
                rB[r] = ts_load4_at<T>(Bp + (int64_t)base * (int32_t)p.B_t, (k * (uint32_t)(int32_t)p.B_t + (uint32_t)bc_at) * (uint32_t)sizeof(T));
                if (second) rC[r] = ts_load4_at<T>(Cp + (int64_t)base * (int32_t)p.C_t, (k * (uint32_t)(int32_t)p.C_t + (uint32_t)bc_at) * (uint32_t)sizeof(T));
            }
            return;
        }
#pragma unroll
        for (int r = 0; r < L::kRounds; ++r) {
            const int64_t k = max(min(base + r * L::kRows + l.row, e - 1), a);
            ru[r] = ts_load4<T>(u + at + k * p.u_t, mine, whole);
            rd[r] = ts_load4<T>(dl + at + k * p.dl_t, mine, whole);
            if (second) {
                ro[r] = ts_load4<T>(dout + at + k * q.do_t, mine, whole);
                if (z) rz[r] = ts_load4<T>(z + at + k * p.z_t, mine, whole);
            }
        }
#pragma unroll
        for (int r = 0; r < L::kBcRounds; ++r) {
            const int64_t k = max(min(base + r * L::kBcRows + l.bc_row, e - 1), a);
            rB[r] = ts_load4<T>(Bp + k * p.B_t + bc_at, bc_n, bc_whole);
            if (second) rC[r] = ts_load4<T>(Cp + k * p.C_t + bc_at, bc_n, bc_whole);
        }
    };
    auto piece_before = [&](int e) {
        TsPiece x;
        x.sp = kPacked ? ts_span_at(ts_rare_args()->f.cu, ts_rare_args()->f.n_seqs, p.tokens, b, e - 1) : TsSpan{b, 0, p.tokens};
        x.a = max(max(x.sp.lo, s0), (e - 1) & ~(kKeep - 1));
        x.e = e;
        return x;
    };
    auto tile_of = [](int t) { return t & ~(kTsTile - 1); };
    auto begin = [&](const TsPiece &x) {                             // the first tile of a piece, and the state before it
        if (!works) return;
        request(tile_of(x.a), x.a, x.e, tile_of(x.a) == tile_of(x.e - 1));
        ts_read_state<kSets, kM>(x.a == x.sp.lo ? of_seq(ts_rare_args()->f.initial, x.sp.seq) : ts_rare_args()->f.kept + (((int64_t)b * ts_rare_args()->f.n_kept + x.a / kKeep) * p.dim + d) * N, N, l, there, next_h);
    };
    auto put_bc = [&](float *to, const Raw4<T> &raw, int k, bool in) {
        float v[4];
        ts_widen<T>(raw, v);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = in && bc_n > 0 ? v[i] : 0.0f;
        *reinterpret_cast<float4 *>(to + k * L::kStates + 4 * l.piece) = make_float4(v[0], v[1], v[2], v[3]);
    };
    // steps of a lane's four channels; 0 outside
    auto steps = [&](const Raw4<T> &raw, bool in, float (&step)[4], float (&slope)[4]) {
        float dv[4];
        ts_widen<T>(raw, dv);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            step[i] = p.softplus ? softplus_log2(fmaf(dv[i], kLog2e, bias[i] * kLog2e)) : dv[i] + bias[i];
            slope[i] = p.softplus ? bwd_sigmoid(dv[i], bias[i]) : 1.0f;
            step[i] = in && (whole || i < mine) ? step[i] : 0.0f;
        }
    };
    // one token of every state of a lane, from step and step u in LDS
    auto forwards = [&](int k, floatx4_t (&h)[kM]) {
        const float2 pair = *reinterpret_cast<const float2 *>(s_tok + k * kRow + 4 * l.chan);
#pragma unroll
        for (int m = 0; m < kM; ++m) {
            floatx4_t kept;
#pragma unroll
            for (int v = 0; v < 4; ++v) kept[v] = __builtin_amdgcn_exp2f(pair.x * A2[m][v]) * h[m][v];
            h[m] = cleared(ts_outer(s_B[k * L::kStates + l.state(m) + l.col], pair.y, kept), m);
        }
    };

    // the memory of a workgroup's sums over channels from token t on
    auto sums_at = [&](int t) { return ts_rare_args()->pBC + ((((int64_t)wg * p.batch + b) * p.tokens + t) * p.groups + g) * N * 2; };
    const int64_t bc_row = (int64_t)p.groups * N * 2;
    auto nothing = [&](int from, int to) {                           // tokens of no sequence: behind the last one and before the first
        const float zeros[4] = {0, 0, 0, 0};
        for (int k = from + l.row; works && k < to; k += L::kRows) {
            ts_store4<T, true>(du + (int64_t)k * p.dim + at, mine, whole, zeros);
            ts_store4<T, true>(dd + (int64_t)k * p.dim + at, mine, whole, zeros);
            if (z) ts_store4<T, true>(dz + (int64_t)k * p.dim + at, mine, whole, zeros);
        }
        float *sums = sums_at(from);
        for (int64_t i = threadIdx.x; i < (int64_t)(to - from) * N * 2; i += kThreads) sums[i / (N * 2) * bc_row + i % (N * 2)] = 0.0f;
    };
    int rest = s1;                                                   // tokens that are still to be walked, s0 .. rest - 1
    if (kPacked) {
        for (TsSpan sp; rest > s0 && (sp = ts_span_at(ts_rare_args()->f.cu, ts_rare_args()->f.n_seqs, p.tokens, b, rest - 1)).seq < 0;) {
            nothing(max(sp.lo, s0), rest);
            rest = max(sp.lo, s0);
        }
    }
    TsPiece now;
    if (rest > s0) {
        now = piece_before(rest);
        begin(now);
    }
    for (int turn = 0; rest > s0; turn ^= kTurns - 1) {
        const int a = now.a, e = now.e;
        const TsSpan sp = now.sp;
        ts_keep_together(e - s0, s1 - s0);
        rest = a;
        TsPiece next = now;
        if (rest > s0) next = piece_before(rest);
        if (kPacked && next.sp.seq < 0) {
            nothing(s0, rest);
            rest = s0;
        }
        const bool more = rest > s0;
        float *s_slot = s_slot_all[turn][wave];
        if (works) {
            if (e == sp.hi) ts_read_state<kSets, kM>(of_seq(ts_rare_args()->dfinal, sp.seq), N, l, there, ga);
            else if (e == s1) ts_read_state<kSets, kM>(ts_rare_args()->behind + (((int64_t)b * ts_rare_args()->slots + seg * ts_rare_args()->each) * p.dim + d) * N, N, l, there, ga);
            const int low = tile_of(a), high = tile_of(e - 1);
            floatx4_t h[kM];
#pragma unroll
            for (int m = 0; m < kM; ++m) h[m] = next_h[m];
            auto slot_of = [&](int t) { return s_slot + t / kTsSub % kSlots * kSlot; };
            auto keep = [&](int t) {
#pragma unroll
                for (int m = 0; m < kM; ++m) *reinterpret_cast<floatx4_t *>(slot_of(t) + (m * kWave + l.lane) * 4) = h[m];
            };
            // ---- forwards over all tiles but the last: the states before every eighth token ------------------------------------------
            for (int base = low; kM > 1 && base < high; base += kTsTile) {
#pragma unroll
                for (int r = 0; r < L::kRounds; ++r) {
                    const int k = r * L::kRows + l.row;
                    const bool in = base + k >= a && base + k < e;
                    float uv[4], step[4], slope[4];
                    ts_widen<T>(ru[r], uv);
                    steps(rd[r], in, step, slope);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        uv[i] = in && (whole || i < mine) ? uv[i] : 0.0f;
                        *reinterpret_cast<float2 *>(s_tok + k * kRow + 4 * (l.at + i)) = make_float2(step[i], step[i] * uv[i]);
                    }
                }
#pragma unroll
                for (int r = 0; r < L::kBcRounds; ++r) {
                    const int k = r * L::kBcRows + l.bc_row;
                    if (L::kBcRows > kTsTile && k >= kTsTile) continue;
                    put_bc(s_B, rB[r], k, base + k >= a && base + k < e);
                }
                request(base + kTsTile, a, e, base + kTsTile == high);
                __builtin_amdgcn_sched_barrier(0);
                wave_lds_sync();
#pragma unroll
                for (int k = 0; k < kTsTile; ++k) {
                    if (k % kTsSub == 0) keep(base + k);
                    if (!kPacked || base + k >= a) forwards(k, h);
                }
                wave_lds_sync();
            }
            // ---- backwards ---------------------------------------------------------------------------------------------------------
            for (int base = high; base >= low; base -= kTsTile) {
                float slope[L::kRounds][4], through[L::kRounds][4];
#pragma unroll
                for (int r = 0; r < L::kRounds; ++r) {
                    const int k = r * L::kRows + l.row;
                    const bool in = base + k >= a && base + k < e;
                    float uv[4], step[4], ov[4], zv[4];
                    ts_widen<T>(ru[r], uv);
                    ts_widen<T>(ro[r], ov);
                    steps(rd[r], in, step, slope[r]);
                    if (z) ts_widen<T>(rz[r], zv);
                    float *to = s_tok + k * kRow + 4 * l.at;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const bool ok = in && (whole || i < mine);
                        uv[i] = ok ? uv[i] : 0.0f;
                        float gate = 1.0f;
                        through[r][i] = 0.0f;
                        if (z) {
                            const float sig = ts_sigmoid(zv[i]);
                            gate = zv[i] * sig;
                            through[r][i] = ov[i] * (sig * fmaf(zv[i], 1.0f - sig, 1.0f));
                        }
                        *reinterpret_cast<float4 *>(to + 4 * i) = make_float4(step[i], step[i] * uv[i], ok ? ov[i] * gate : 0.0f, uv[i]);
                    }
                }
#pragma unroll
                for (int r = 0; r < L::kBcRounds; ++r) {
                    const int k = r * L::kBcRows + l.bc_row;
                    if (L::kBcRows > kTsTile && k >= kTsTile) continue;
                    put_bc(s_B, rB[r], k, base + k >= a && base + k < e);
                    put_bc(s_C, rC[r], k, base + k >= a && base + k < e);
                }
                if (base > low) request(base - kTsTile, a, e, true);
                else if (more) begin(next);
                __builtin_amdgcn_sched_barrier(0);
                wave_lds_sync();
                if (base == high) {                                  // the last tile's states
                    keep(base);
                    if (base + kTsSub < e) {
#pragma unroll
                        for (int k = 0; k < kTsSub; ++k)
                            if (!kPacked || base + k >= a) forwards(k, h);
                        keep(base + kTsSub);
                    }
                }
                float y[kTsTile];
#pragma unroll
                for (int half = 1; half >= 0; --half) {
                    const int k0 = half * kTsSub;
#pragma unroll
                    for (int i = 0; i < kTsSub; ++i) y[k0 + i] = 0.0f;
                    if (base + k0 >= e || base + k0 + kTsSub <= a) continue;               // uniform
                    float *slot = slot_of(base + k0);
                    float sq[2 * kTsSub];                            // s of the eight tokens, w . A of the eight
#pragma unroll
                    for (int i = 0; i < 2 * kTsSub; ++i) sq[i] = 0.0f;
                    constexpr bool kRepairs = kM < 4;
                    auto there_at = [&](int i) { return base + k0 + i >= a && base + k0 + i < e; };
                    const bool some = kRagged && !(base + k0 >= a && base + k0 + kTsSub <= e);         // of the eight
                    // Of more than 32 states a branch to a token: that kernel waits for registers, which it leaves free (6007 packed tokens of 64 states 2605 -> 1741 us).  Of fewer it
                    // would cost every tile 8 to 14 %: states, decays and dA are found again where some are not there, 4 x 2041 tokens 407 -> 423 us, 12 011 packed 554 -> 560, 2 x 2041
                    // of 32 states 556 -> 587 (637 by branches).
                    auto in = [&](int i) { return !kRagged || kRepairs || there_at(i); };
#pragma unroll
                    for (int m = 0; m < kM; ++m) {
                        floatx4_t hs[kTsSub + 1], decay[kTsSub] = {};
                        hs[0] = *reinterpret_cast<const floatx4_t *>(slot + (m * kWave + l.lane) * 4);
#pragma unroll
                        for (int i = 0; i < kTsSub; ++i) {
                            if (!in(i)) {
                                hs[i + 1] = hs[i];
                                continue;
                            }
                            const float *row = s_tok + (k0 + i) * kRow + 4 * l.chan;
                            const float2 pair = *reinterpret_cast<const float2 *>(row);
                            floatx4_t kept;
#pragma unroll
                            for (int v = 0; v < 4; ++v) {
                                decay[i][v] = __builtin_amdgcn_exp2f(pair.x * A2[m][v]);
                                kept[v] = decay[i][v] * hs[i][v];
                            }
                            hs[i + 1] = cleared(ts_outer(s_B[(k0 + i) * L::kStates + l.state(m) + l.col], pair.y, kept), m);
                        }
                        floatx4_t dA_some = {0, 0, 0, 0};
                        if (kRepairs && some) {                       // states, decays and dA again, of its tokens alone
#pragma unroll
                            for (int i = 0; i < kTsSub; ++i) {
                                if (!there_at(i)) {
                                    hs[i + 1] = hs[i];
                                    decay[i] = floatx4_t{1, 1, 1, 1};
                                    continue;
                                }
                                const float2 pair = *reinterpret_cast<const float2 *>(s_tok + (k0 + i) * kRow + 4 * l.chan);
                                floatx4_t kept;
#pragma unroll
                                for (int v = 0; v < 4; ++v) kept[v] = decay[i][v] * hs[i][v];
                                hs[i + 1] = cleared(ts_outer(s_B[(k0 + i) * L::kStates + l.state(m) + l.col], pair.y, kept), m);
                            }
                            floatx4_t g_at = ga[m];
                            dA_some = dA[m];
#pragma unroll
                            for (int i = kTsSub - 1; i >= 0; --i) {
                                if (!there_at(i)) continue;
                                const float4 tok = *reinterpret_cast<const float4 *>(s_tok + (k0 + i) * kRow + 4 * l.chan);
                                const floatx4_t gr = cleared(ts_outer(s_C[(k0 + i) * L::kStates + l.state(m) + l.col], tok.z, g_at), m);
#pragma unroll
                                for (int v = 0; v < 4; ++v) {
                                    g_at[v] = decay[i][v] * gr[v];
                                    dA_some[v] = fmaf(g_at[v] * hs[i][v], tok.x, dA_some[v]);
                                }
                            }
                        }
                        if (z) {
#pragma unroll
                            for (int i = 0; i < kTsSub; ++i) {
                                const float4 c = *reinterpret_cast<const float4 *>(s_C + (k0 + i) * L::kStates + l.state(m));
                                y[k0 + i] = fmaf(c.w, hs[i + 1][3], fmaf(c.z, hs[i + 1][2], fmaf(c.y, hs[i + 1][1], fmaf(c.x, hs[i + 1][0], y[k0 + i]))));
                            }
                        }
#pragma unroll
                        for (int two = kTsSub / 2 - 1; two >= 0; --two) {
                            float both[16];
#pragma unroll
                            for (int par = 1; par >= 0; --par) {
                                const int i = 2 * two + par;
                                if (!in(i)) {
#pragma unroll
                                    for (int v = 0; v < 8; ++v) both[8 * par + v] = 0.0f;
                                    continue;
                                }
                                const float4 tok = *reinterpret_cast<const float4 *>(s_tok + (k0 + i) * kRow + 4 * l.chan);
                                const floatx4_t gr = cleared(ts_outer(s_C[(k0 + i) * L::kStates + l.state(m) + l.col], tok.z, ga[m]), m);
                                const float4 Bv = *reinterpret_cast<const float4 *>(s_B + (k0 + i) * L::kStates + l.state(m));
                                sq[i] = fmaf(gr[3], Bv.w, fmaf(gr[2], Bv.z, fmaf(gr[1], Bv.y, fmaf(gr[0], Bv.x, sq[i]))));
#pragma unroll
                                for (int v = 0; v < 4; ++v) {
                                    both[8 * par + v] = tok.y * gr[v];
                                    both[8 * par + 4 + v] = tok.z * hs[i + 1][v];
                                    ga[m][v] = decay[i][v] * gr[v];
                                    const float w = ga[m][v] * hs[i][v];
                                    dA[m][v] = fmaf(w, tok.x, dA[m][v]);
                                    sq[kTsSub + i] = fmaf(w, A2[m][v], sq[kTsSub + i]);
                                }
                            }
                            const float total = ts_sum_channels<kSets>(both, l.lane);
                            const int par = l.lane >> 5, is_c = l.lane >> 4 & 1, v = l.lane & 3;
                            slot[m * 4 * kWave + ((2 * two + par) * kQuarter + 4 * l.set + v) * 2 + is_c] = total;
                        }
                        if (kRepairs && some) dA[m] = dA_some;
                    }
                    wave_lds_sync();
                    ts_sum_sets<kSets>(sq);
                    constexpr int kLeft = 16 / kSets;
#pragma unroll
                    for (int i = 0; i < kLeft; ++i) {
                        const int entry = kLeft * l.set + i, row = k0 + entry % kTsSub;
                        *(entry < kTsSub ? s_tok + row * kRow + 4 * l.chan + 1 : s_q + row * L::kPitch + l.chan) = sq[i];
                    }
                }
                if (z) {
                    ts_sum_sets<kSets>(y);
                    constexpr int kLeft = 16 / kSets;
#pragma unroll
                    for (int i = 0; i < kLeft; ++i) s_y[(kLeft * l.set + i) * L::kPitch + l.chan] = y[i];
                }
                wave_lds_sync();
#pragma unroll
                for (int r = 0; r < L::kRounds; ++r) {
                    const int k = r * L::kRows + l.row;
                    if (base + k < a || base + k >= e) continue;
                    auto row_of = [&](T *t) {
                        if constexpr (kQuick) return reinterpret_cast<T *>(reinterpret_cast<char *>(t + (int64_t)base * p.dim) + ((uint32_t)k * (uint32_t)p.dim + (uint32_t)at) * (uint32_t)sizeof(T));
                        return t + (int64_t)(base + k) * p.dim + at;
                    };
                    const float4 q4 = *reinterpret_cast<const float4 *>(s_q + k * L::kPitch + l.at);
                    const float qv[4] = {q4.x, q4.y, q4.z, q4.w};
                    float u_out[4], d_out[4], uv[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float4 tok = *reinterpret_cast<const float4 *>(s_tok + k * kRow + 4 * (l.at + i));       // step, s, dy, u
                        uv[i] = tok.w;
                        u_out[i] = p.D ? fmaf(skip[i], tok.z, tok.x * tok.y) : tok.x * tok.y;
                        d_out[i] = fmaf(kLn2, qv[i], tok.w * tok.y) * slope[r][i];
                        sum_bias[i] += d_out[i];
                        sum_D[i] = fmaf(tok.z, tok.w, sum_D[i]);
                    }
                    ts_store4<T, true>(row_of(du), mine, whole, u_out);
                    ts_store4<T, true>(row_of(dd), mine, whole, d_out);
                    if (z) {
                        const float4 y4 = *reinterpret_cast<const float4 *>(s_y + k * L::kPitch + l.at);
                        const float yv[4] = {y4.x, y4.y, y4.z, y4.w};
#pragma unroll
                        for (int i = 0; i < 4; ++i) u_out[i] = through[r][i] * (p.D ? fmaf(skip[i], uv[i], yv[i]) : yv[i]);
                        ts_store4<T, true>(row_of(dz), mine, whole, u_out);
                    }
                }
                wave_lds_sync();
            }
            if (a == sp.lo && ts_rare_args()->dinitial) ts_write_state<kSets, kM>(ts_rare_args()->dinitial + ((int64_t)sp.seq * p.dim + d) * N, N, l, there, ga);
        }
        // ---- the piece's dB and dC over the workgroup's channels ---------------------------------------------------------------------
        __syncthreads();
        float *pBC = sums_at(a);
        for (int i = threadIdx.x; i < (e - a) * L::kStates * 2; i += kThreads) {
            const int k = i / (2 * L::kStates), n = i % (2 * L::kStates) / 2, c = i & 1, t = a + k;
            const int from = t / kTsSub % kSlots * kSlot + n / kQuarter * 4 * kWave + (t % kTsSub * kQuarter + n % kQuarter) * 2 + c;
            float total = 0.0f;
            for (int w = 0; w < n_works; ++w) total += s_slot_all[turn][w][from];
            if (n < N) pBC[(int64_t)k * bc_row + 2 * n + c] = total;
        }
        if constexpr (kTurns == 1) __syncthreads();                  // (with two, the next piece's barrier comes before these are written again)
        now = next;
    }
    if (!works) return;
    const int64_t part = (int64_t)b * p.n_segs + seg;
    ts_write_state<kSets, kM>(ts_rare_args()->pA + (part * p.dim + d) * N, N, l, there, dA);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int over = L::kCols; over < kWave; over *= 2) {
            sum_D[i] += __shfl_xor(sum_D[i], over, kWave);
            sum_bias[i] += __shfl_xor(sum_bias[i], over, kWave);
        }
        if (l.row == 0 && i < mine) {
            ts_rare_args()->pD[part * 2 * p.dim + c0 + at + i] = sum_D[i];
            ts_rare_args()->pD[(part * 2 + 1) * p.dim + c0 + at + i] = sum_bias[i];
        }
    }
}

// dB and dC: over the workgroups of a group
template <typename T> __global__ __launch_bounds__(kBlock) void ts_sum_bc_kernel(const float2 *__restrict__ from, T *__restrict__ dB, T *__restrict__ dC, int64_t n, int parts) {
    const int64_t i = (int64_t)blockIdx.x * kBlock + threadIdx.x;
    if (i >= n) return;
    float2 total = from[i];
    for (int k = 1; k < parts; ++k) {
        const float2 v = from[k * n + i];
        total.x += v.x;
        total.y += v.y;
    }
    dB[i] = from_f32<T>(total.x);
    dC[i] = from_f32<T>(total.y);
}

// dA, dD and the bias's gradient: over rows and segments; a thread per value of (channel, state), then D and bias
static __global__ __launch_bounds__(kBlock) void ts_sum_rows_kernel(const float *__restrict__ pA, const float *__restrict__ pD, float *dA, float *dD, float *dbias, int dim, int n_A, int parts) {
    const uint32_t i = blockIdx.x * kBlock + threadIdx.x;
    if (i >= (uint32_t)n_A + 2u * (uint32_t)dim) return;
    const bool is_A = i < (uint32_t)n_A;
    const uint32_t j = i - (uint32_t)n_A;
    const int64_t pitch = is_A ? n_A : 2 * (int64_t)dim;
    const float *from = is_A ? pA + i : pD + j;
    float *to = is_A ? dA : j < (uint32_t)dim ? dD : dbias;
    if (!to) return;
    float total[4] = {0, 0, 0, 0};
    int k = 0;
    for (; k + 4 <= parts; k += 4)
#pragma unroll
        for (int e = 0; e < 4; ++e) total[e] += from[(k + e) * pitch];
    for (; k < parts; ++k) total[0] += from[k * pitch];
    to[is_A ? i : j % (uint32_t)dim] = (total[0] + total[1]) + (total[2] + total[3]);
}

// ---- launches, one type to a source (token_scan_bwd_*.hip) ----------------------------------------------------------------------------
template <typename T> int ts_bwd_run(const ss2d_token_scan_bwd_params *p, const TsBwdArgs &q, hipStream_t st) {
    using std::integral_constant;
    const TsArgs &a = q.f;
    auto run_as = [&](auto sets, auto m, auto quick, auto ends) {
        constexpr int kSets = decltype(sets)::value, kM = decltype(m)::value;
        constexpr bool kQuick = decltype(quick)::value;
        constexpr TsEnds kEnds = decltype(ends)::value;
        if (a.n_segs > 1) {
            TsBwdArgs left = q;
            left.f.wgs = q.left_wgs;
            left.f.seg_len = a.seg_len / q.each;
            ts_left_kernel<T, kSets, kM, kQuick><<<(uint32_t)(a.batch * a.groups * q.left_wgs * q.slots), kBlock, 0, st>>>(left);
            const uint32_t per_row = (uint32_t)a.dim * a.N;
            ts_join_left_kernel<<<dim3((per_row + kBlock - 1) / kBlock, a.batch), kBlock, 0, st>>>(q, per_row);
        }
        ts_grad_kernel<T, kSets, kM, kQuick, kEnds><<<(uint32_t)(a.batch * a.groups * a.wgs * a.n_segs), kWave * kTsBwdWaves<kM>, 0, st>>>(q);
    };
    auto run = [&](auto sets, auto m) {
        auto by_ends = [&](auto quick) {
            if (a.cu) run_as(sets, m, quick, integral_constant<TsEnds, kTsPacked>{});
            else if (a.tokens % kTsSub) run_as(sets, m, quick, integral_constant<TsEnds, kTsLast>{});
            else run_as(sets, m, quick, integral_constant<TsEnds, kTsWhole>{});
        };
        ts_quick(a) ? by_ends(std::true_type{}) : by_ends(std::false_type{});
    };
    if (a.N <= 4) run(integral_constant<int, 1>{}, integral_constant<int, 1>{});
    else if (a.N <= 8) run(integral_constant<int, 2>{}, integral_constant<int, 1>{});
    else if (a.N <= 16) run(integral_constant<int, 4>{}, integral_constant<int, 1>{});
    else if (a.N <= 32) run(integral_constant<int, 4>{}, integral_constant<int, 2>{});
    else run(integral_constant<int, 4>{}, integral_constant<int, 4>{});
    const int64_t n = (int64_t)a.batch * a.tokens * a.groups * a.N;
    ts_sum_bc_kernel<T><<<(uint32_t)((n + kBlock - 1) / kBlock), kBlock, 0, st>>>((const float2 *)q.pBC, (T *)p->dB, (T *)p->dC, n, a.wgs);
    const int n_A = a.dim * a.N;
    if (p->dA || p->dD || p->ddelta_bias)
        ts_sum_rows_kernel<<<(uint32_t)((n_A + 2 * (int64_t)a.dim + kBlock - 1) / kBlock), kBlock, 0, st>>>(q.pA, q.pD, p->dA, p->dD, p->ddelta_bias, a.dim, n_A, a.batch * a.n_segs);
    return launch_status();
}

}  // namespace ss2d
