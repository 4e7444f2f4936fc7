// Forward of the selective scan of token sequences (token_scan.h).
//
// A tile of 16 tokens: the lanes take four channels of a token each, find step, step u and the skip term, and lay step and step u down in LDS; B and C
// come as fp32 rows beside them.  Then every lane walks the 16 tokens of its channel's states; the sums C . h of the sets meet in DPP additions, go through LDS back to
// the lanes of the first kind, which add the skip term, apply the gate and store.  The next tile's loads are on their way meanwhile.  A wavefront meets no
// other: no workgroup barrier.
//
// Vector instructions bound it: 421 for a tile of 4096 values of states, 80 of them exponentials and the like of twice the time; they are issued in 96 % of the CUs' busy cycles.  32768 tokens of 2048
// channels, 16 states, bf16: 236 us, and 170 for what 31 of 32 segments leave (without the sums, gates and outputs, 286 a tile, 92 %); one pass over the states of the same
// length, without segments, would keep an eighth of the SIMDs busy.  Where wavefronts run as they come the last ones end alone: 266 and 198 us, 83 % and 79 % (ts_keep_together).
#include "token_scan.h"

namespace ss2d {

// kLocal: what a segment leaves, instead of its outputs.  kQuick: see ts_quick.
template <typename T, int kSets, int kM, bool kLocal, bool kQuick>
__global__ __launch_bounds__(kBlock, kM == 4 ? 2 : 3) void ts_kernel(const TsArgs p) {
    using L = TsLane<kSets, kM>;
    __shared__ __align__(16) float s_all[kWavesPerWg][kTsTile * (L::kPairPitch + 2 * L::kStates)];
    const L l(threadIdx.x & (kWave - 1));
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    float *s_step = s_all[wave], *s_B = s_step + kTsTile * L::kPairPitch, *s_C = s_B + kTsTile * L::kStates, *s_y = s_step;
    uint32_t id = xcd_contiguous_id(blockIdx.x, gridDim.x);
    const int wg = (int)(id % (uint32_t)p.wgs); id /= (uint32_t)p.wgs;
    const int g = (int)(id % (uint32_t)p.groups); id /= (uint32_t)p.groups;
    const int segs = kLocal ? p.n_segs - 1 : p.n_segs, seg = (int)(id % (uint32_t)segs), b = (int)(id / (uint32_t)segs);
    const int first = (wg * kWavesPerWg + wave) * L::kCh, n_chan = min(L::kCh, p.per_group - first);
    if (n_chan <= 0) return;
    const int c0 = g * p.per_group + first, s0 = seg * p.seg_len, s1 = s0 + min(p.seg_len, p.tokens - s0);
    const bool whole = kQuick || n_chan == L::kCh;
    const int mine = kQuick ? 4 : min(max(n_chan - l.at, 0), 4);                  // channels of a lane that stages
    const int at = mine > 0 ? l.at : 0;
    const bool there = kQuick || l.chan < n_chan;
    const int d = c0 + (kQuick ? l.chan : min(l.chan, n_chan - 1));
    const int N = kQuick ? L::kStates : p.N;

    int t = s0;
    TsSpan sp = {b, 0, p.tokens};
    int64_t state_at = 0;
    if constexpr (kLocal) {
        sp = ts_span_at(p.cu, p.n_seqs, p.tokens, b, s1 - 1);
        const int carry = sp.seq < 0 || sp.hi <= s1 ? kTsNothing : sp.lo >= s0 ? kTsStarts : kTsThrough;
        if (wg == 0 && g == 0 && threadIdx.x == 0) p.flags[(int64_t)b * segs + seg] = carry;
        if (carry == kTsNothing) return;
        t = max(s0, sp.lo);
        state_at = (((int64_t)b * segs + seg) * p.dim + d) * N;
    } else {
        sp = ts_span_at(p.cu, p.n_seqs, p.tokens, b, t);
    }

    const T *Bp = (const T *)p.B + (int64_t)b * p.B_b + (int64_t)g * p.B_g, *Cp = (const T *)p.C + (int64_t)b * p.C_b + (int64_t)g * p.C_g;
    T *out = (T *)p.out + (int64_t)b * p.tokens * p.dim + c0 + at;
    const int bc_n = kQuick ? 4 : min(max(N - 4 * l.piece, 0), 4), bc_at = bc_n > 0 ? 4 * l.piece : 0;
    const bool bc_whole = kQuick || N == L::kStates;
    float bias[4], bias2[4], skip[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        bias[i] = p.bias && i < mine ? p.bias[c0 + at + i] : 0.0f;
        bias2[i] = bias[i] * kLog2e;
        skip[i] = p.D && i < mine ? p.D[c0 + at + i] : 0.0f;
    }
    floatx4_t A2[kM], h[kM];
    ts_read_state<kSets, kM>(p.A + (int64_t)d * N, N, l, true, A2);
#pragma unroll
    for (int m = 0; m < kM; ++m) A2[m] *= kLog2e;
    auto start = [&](const TsSpan &s) { ts_read_state<kSets, kM>(p.initial ? p.initial + ((int64_t)s.seq * p.dim + d) * N : nullptr, N, l, there, h); };
    auto nothing = [&](int from, int to) {                           // tokens of no sequence
        if constexpr (!kLocal) {
            const float zeros[4] = {0, 0, 0, 0};
            for (int k = from + l.row; k < to; k += L::kRows) ts_store4<T>(out + (int64_t)k * p.dim, mine, whole, zeros);
        }
    };
    if constexpr (!kLocal) {
        if (p.cu && p.final)                                         // sequences without tokens, dealt out over the segments
            for (uint32_t i = seg; i < (uint32_t)p.n_seqs; i += p.n_segs) {
                const int lo = min(max(p.cu[i], 0), p.tokens), hi = min(max(p.cu[i + 1], 0), p.tokens);
                if (hi > lo) continue;
                start({(int)i, lo, lo});
                ts_write_state<kSets, kM>(p.final + ((int64_t)i * p.dim + d) * N, N, l, there, h);
            }
        while (sp.seq < 0) {
            nothing(t, min(sp.hi, s1));
            t = sp.hi;
            if (t >= s1) return;
            sp = ts_span_at(p.cu, p.n_seqs, p.tokens, b, t);
        }
    }
    if (t == sp.lo) start(sp);
    else if constexpr (kLocal) {
#pragma unroll
        for (int m = 0; m < kM; ++m) h[m] = floatx4_t{0, 0, 0, 0};
    } else {
        ts_read_state<kSets, kM>(p.enter + (((int64_t)b * (p.n_segs - 1) + seg - 1) * p.dim + d) * N, N, l, there, h);
    }

    Raw4<T> ru[L::kRounds], rd[L::kRounds], rz[L::kRounds], rB[L::kBcRounds], rC[L::kBcRounds];
    // tokens from .. to - 1 of one tile
    const T *u0 = (const T *)p.u + (int64_t)b * p.u_b + c0, *dl0 = (const T *)p.delta + (int64_t)b * p.dl_b + c0, *z0 = p.z ? (const T *)p.z + (int64_t)b * p.z_b + c0 : nullptr;
    T *out0 = (T *)p.out + (int64_t)b * p.tokens * p.dim + c0;
    auto request = [&](int from, int to) {
        if constexpr (kQuick) {                                      // (a uniform base, and 32 bits from there on)
            auto row_of = [&](int k) { return (uint32_t)min(k, to - 1 - from); };
#pragma unroll
            for (int r = 0; r < L::kRounds; ++r) {
                const uint32_t k = row_of(r * L::kRows + l.row);
                ru[r] = ts_load4_at<T>(u0 + from * p.u_t, (k * (uint32_t)p.u_t + (uint32_t)at) * (uint32_t)sizeof(T));
                rd[r] = ts_load4_at<T>(dl0 + from * p.dl_t, (k * (uint32_t)p.dl_t + (uint32_t)at) * (uint32_t)sizeof(T));
                if constexpr (!kLocal) if (z0) rz[r] = ts_load4_at<T>(z0 + from * p.z_t, (k * (uint32_t)p.z_t + (uint32_t)at) * (uint32_t)sizeof(T));
            }
#pragma unroll
            for (int r = 0; r < L::kBcRounds; ++r) {
                const uint32_t k = row_of(r * L::kBcRows + l.bc_row);
                rB[r] = ts_load4_at<T>(Bp + from * p.B_t, (k * (uint32_t)p.B_t + (uint32_t)bc_at) * (uint32_t)sizeof(T));
                if constexpr (!kLocal) rC[r] = ts_load4_at<T>(Cp + from * p.C_t, (k * (uint32_t)p.C_t + (uint32_t)bc_at) * (uint32_t)sizeof(T));
            }
            return;
        }
#pragma unroll
        for (int r = 0; r < L::kRounds; ++r) {
            const int64_t k = min(from + r * L::kRows + l.row, to - 1);
            ru[r] = ts_load4<T>(u0 + at + k * p.u_t, mine, whole);
            rd[r] = ts_load4<T>(dl0 + at + k * p.dl_t, mine, whole);
            if constexpr (!kLocal) if (z0) rz[r] = ts_load4<T>(z0 + at + k * p.z_t, mine, whole);
        }
#pragma unroll
        for (int r = 0; r < L::kBcRounds; ++r) {
            const int64_t k = min(from + r * L::kBcRows + l.bc_row, to - 1);
            rB[r] = ts_load4<T>(Bp + k * p.B_t + bc_at, bc_n, bc_whole);
            if constexpr (!kLocal) rC[r] = ts_load4<T>(Cp + k * p.C_t + bc_at, bc_n, bc_whole);
        }
    };
    auto tile_end = [&](int from, const TsSpan &s) { return min(min(s.hi, s1), (from | (kTsTile - 1)) + 1); };
    float sum[4] = {0, 0, 0, 0};                                     // kLocal: the steps of a lane's tokens and channels
    int end = tile_end(t, sp);
    request(t, end);
    for (;;) {
        const int n = end - t;
        ts_keep_together(s1 - t, s1 - s0);
        // ---- stage -----------------------------------------------------------------------------------------------------------
        float extra[L::kRounds][4], gate[L::kRounds][4];
        auto stage = [&](auto all) {                                 // all: 16 tokens, every lane's channels and states there
            constexpr bool kAll = decltype(all)::value;
#pragma unroll
            for (int r = 0; r < L::kRounds; ++r) {
                const int k = r * L::kRows + l.row;
                float uv[4], dv[4], step[4];
                ts_widen<T>(ru[r], uv);
                ts_widen<T>(rd[r], dv);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    step[i] = p.softplus ? softplus_log2(fmaf(dv[i], kLog2e, bias2[i])) : dv[i] + bias[i];
                    if constexpr (!kAll) {
                        const bool in = k < n && (whole || i < mine);
                        step[i] = in ? step[i] : 0.0f;
                        uv[i] = in ? uv[i] : 0.0f;
                    }
                    extra[r][i] = p.D ? skip[i] * uv[i] : 0.0f;      // (without D no term: an infinite u would make 0 u of it)
                    if constexpr (kLocal) sum[i] += step[i];
                }
                float *to = s_step + k * L::kPairPitch + 2 * l.at;
                *reinterpret_cast<float4 *>(to) = make_float4(step[0], step[0] * uv[0], step[1], step[1] * uv[1]);
                *reinterpret_cast<float4 *>(to + 4) = make_float4(step[2], step[2] * uv[2], step[3], step[3] * uv[3]);
                if constexpr (!kLocal) {
                    if (z0) {
                        float zv[4];
                        ts_widen<T>(rz[r], zv);
#pragma unroll
                        for (int i = 0; i < 4; ++i) gate[r][i] = zv[i] * ts_sigmoid(zv[i]);
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; ++i) gate[r][i] = 1.0f;
                    }
                }
            }
#pragma unroll
            for (int r = 0; r < L::kBcRounds; ++r) {
                const int k = r * L::kBcRows + l.bc_row;
                if (L::kBcRows > kTsTile && k >= kTsTile) continue;
                auto put = [&](float *to, const Raw4<T> &raw) {
                    float v[4];
                    ts_widen<T>(raw, v);
                    if constexpr (!kAll)
#pragma unroll
                        for (int i = 0; i < 4; ++i) v[i] = k < n && bc_n > 0 ? v[i] : 0.0f;
                    *reinterpret_cast<float4 *>(to + k * L::kStates + 4 * l.piece) = make_float4(v[0], v[1], v[2], v[3]);
                };
                put(s_B, rB[r]);
                if constexpr (!kLocal) put(s_C, rC[r]);
            }
        };
        if (kQuick && n == kTsTile) stage(std::true_type{});
        else stage(std::false_type{});
        // ---- the next tile, and what it starts with -----------------------------------------------------------------------------
        const int next = end;
        const bool ends = next == sp.hi;                             // (of the sequence)
        const TsSpan was = sp;
        int next_end = next, zeros_to = 0;
        if (next < s1) {
            if (ends) sp = ts_span_at(p.cu, p.n_seqs, p.tokens, b, next);
            if (sp.seq < 0) zeros_to = min(sp.hi, s1);               // (behind the last sequence)
            else next_end = tile_end(next, sp);
        }
        if (next_end > next) request(next, next_end);
        __builtin_amdgcn_sched_barrier(0);
        wave_lds_sync();
        // ---- compute ---------------------------------------------------------------------------------------------------------
        if constexpr (!kLocal) {
            if (p.kept && (t & (p.keep - 1)) == 0 && t > 0)
                ts_write_state<kSets, kM>(p.kept + (((int64_t)b * p.n_kept + t / p.keep) * p.dim + d) * N, N, l, there, h);
        }
        float y[kTsTile];
        // tokens: the tile has its 16 (those it has not are not walked: a step of 0 is none to an A of -inf); states: every value of a lane is one.  One walk of both kinds of tiles, and
        // the states behind it put right, is no faster (32768 tokens 416 us, this 414) and of 64 states 6.4 ms where this is 0.72.
        auto walk = [&](auto tokens, auto states) {
            constexpr bool kTokens = decltype(tokens)::value, kStates = decltype(states)::value;
#pragma unroll
            for (int k = 0; k < kTsTile; ++k) {
                y[k] = 0.0f;
                if (!kTokens && k >= n) continue;                       // (uniform)
                const float2 pair = *reinterpret_cast<const float2 *>(s_step + k * L::kPairPitch + 2 * l.chan);
#pragma unroll
                for (int m = 0; m < kM; ++m) {
                    floatx4_t kept;
#pragma unroll
                    for (int v = 0; v < 4; ++v) kept[v] = __builtin_amdgcn_exp2f(pair.x * A2[m][v]) * h[m][v];
                    h[m] = ts_outer(s_B[k * L::kStates + l.state(m) + l.col], pair.y, kept);
                    if constexpr (!kLocal) {
                        if constexpr (!kStates) ts_clear_others<kSets, kM>(h[m], m, N, l, true);
                        const float4 c = *reinterpret_cast<const float4 *>(s_C + k * L::kStates + l.state(m));
                        y[k] = fmaf(c.w, h[m][3], fmaf(c.z, h[m][2], fmaf(c.y, h[m][1], fmaf(c.x, h[m][0], y[k]))));
                    }
                }
            }
        };
        constexpr std::bool_constant<kQuick || kLocal> quick;
        if (n != kTsTile) walk(std::false_type{}, quick);
        else if (quick.value || bc_whole) walk(std::true_type{}, std::true_type{});
        else walk(std::true_type{}, quick);
        wave_lds_sync();
        if constexpr (!kLocal) {
            ts_sum_sets<kSets>(y);
            constexpr int kLeft = kTsTile / kSets;
#pragma unroll
            for (int i = 0; i < kLeft; ++i) s_y[(kLeft * l.set + i) * L::kPitch + l.chan] = y[i];
            wave_lds_sync();
#pragma unroll
            for (int r = 0; r < L::kRounds; ++r) {
                const int k = r * L::kRows + l.row;
                const float4 part = *reinterpret_cast<const float4 *>(s_y + k * L::kPitch + l.at);
                const float o[4] = {(part.x + extra[r][0]) * gate[r][0], (part.y + extra[r][1]) * gate[r][1], (part.z + extra[r][2]) * gate[r][2],
                                    (part.w + extra[r][3]) * gate[r][3]};
                if (k >= n) continue;
                if constexpr (kQuick) ts_store4<T>(reinterpret_cast<T *>(reinterpret_cast<char *>(out0 + (int64_t)t * p.dim) + ((uint32_t)k * (uint32_t)p.dim + (uint32_t)at) * (uint32_t)sizeof(T)), 4, true, o);
                else ts_store4<T>(out + (int64_t)(t + k) * p.dim, mine, whole, o);
            }
            wave_lds_sync();
            if (ends && p.final) ts_write_state<kSets, kM>(p.final + ((int64_t)was.seq * p.dim + d) * N, N, l, there, h);
        }
        if (next_end == next) {
            nothing(next, zeros_to);
            break;
        }
        if (ends) start(sp);
        t = next;
        end = next_end;
    }
    if constexpr (kLocal) {
        ts_write_state<kSets, kM>(p.end + state_at, N, l, there, h);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
            for (int over = L::kCols; over < kWave; over *= 2) sum[i] += __shfl_xor(sum[i], over, kWave);
            if (l.row == 0 && i < mine) p.sums[((int64_t)b * segs + seg) * p.dim + c0 + at + i] = sum[i];
        }
    }
}

// What enters every segment but the first: a thread per (row, channel, state)
__global__ __launch_bounds__(kBlock) void ts_join_kernel(const TsArgs p, uint32_t per_row) {
    const uint32_t item = blockIdx.x * kBlock + threadIdx.x;
    const int b = (int)blockIdx.y, segs = p.n_segs - 1;
    if (item >= per_row) return;
    const uint32_t d = item / (uint32_t)p.N;
    const float A2 = 0.5f * kLog2e * p.A[item];
    const float *end = p.end + (int64_t)b * segs * per_row + item, *sums = p.sums + (int64_t)b * segs * p.dim + d;
    const int32_t *flags = p.flags + (int64_t)b * segs;
    float *enter = p.enter + (int64_t)b * segs * per_row + item;
    constexpr int kFly = 8;
    float carry = 0.0f;
    for (int s0 = 0; s0 < segs; s0 += kFly) {
        float left[kFly], sum[kFly];
        int flag[kFly];
#pragma unroll
        for (int i = 0; i < kFly; ++i) {
            const int s = min(s0 + i, segs - 1);
            left[i] = end[(int64_t)s * per_row];
            sum[i] = sums[(int64_t)s * p.dim];
            flag[i] = flags[s];
        }
#pragma unroll
        for (int i = 0; i < kFly; ++i) {
            if (s0 + i >= segs) break;
            if (flag[i] == kTsThrough && carry != 0.0f) {
                carry = ts_handed_on(carry, A2, sum[i], left[i]);
            } else {
                carry = flag[i] == kTsNothing ? 0.0f : left[i];      // (of nothing, the segment's memory holds nothing)
            }
            enter[(int64_t)(s0 + i) * per_row] = carry;
        }
    }
}

// ---- host ------------------------------------------------------------------------------------------------------------------------
// Segments of the token axis.  A cut sequence is walked twice for what goes into the later segments, so it is cut only where its wavefronts are fewer than one and a half to
// a SIMD, and then into as many as come to four workgroups on every CU: what is between two whole numbers of them waits for the last.  Rows of 4096 tokens of 2048 channels, cut and whole: 8 of them 386 and
// 619 us, 11 637 and 673, 12 (from which on they are left whole) 639 and 673, 14 705 and 679, 16 710 and 680, 24 782 and 781.
static void ts_cut(TsArgs &a) {
    const int ch = kWave / ts_sets(a.N);
    a.wgs = (int)(((int64_t)a.per_group + ch * kWavesPerWg - 1) / (ch * kWavesPerWg));
    const int64_t waves = (int64_t)a.batch * a.groups * ((a.per_group + ch - 1) / ch), wgs = (int64_t)a.batch * a.groups * a.wgs;
    constexpr int64_t kEnough = 1536, kTarget = 1024;
    int64_t n = waves >= kEnough ? 1 : kTarget / (wgs > 0 ? wgs : 1);
    const int64_t most = (a.tokens + 2 * kTsGrid - 1) / (2 * kTsGrid);
    n = n < most ? n : most;
    a.seg_len = ts_seg_len(a.tokens, n, a.keep);
    a.n_segs = (int)((a.tokens + (int64_t)a.seg_len - 1) / a.seg_len);
    if (a.n_segs < 1) a.n_segs = 1;
}

static int64_t ts_carve(TsArgs &a, uint8_t *base) {
    int64_t at = 0;
    auto take = [&](int64_t bytes) { uint8_t *p = base ? base + at : nullptr; at += (bytes + 255) / 256 * 256; return p; };
    const int64_t cuts = (int64_t)a.batch * (a.n_segs - 1);
    a.end = (float *)take(cuts * a.dim * a.N * 4);
    a.enter = (float *)take(cuts * a.dim * a.N * 4);
    a.sums = (float *)take(cuts * a.dim * 4);
    a.flags = (int32_t *)take(cuts * 4);
    return at;
}

int ts_read(const ss2d_token_scan_params *p, TsArgs &a) {
    a = {};
    if (!p || p->batch < 0 || p->seqlen < 0 || p->dim < 0 || p->dstate < 1 || p->n_groups < 1 || p->n_seqs < 0) return SS2D_EINVAL;
    if (p->dtype < SS2D_F32 || p->dtype > SS2D_F16 || p->dim % p->n_groups) return SS2D_EINVAL;
    if (p->cu_seqlens && (p->batch != 1 || p->n_seqs < 1)) return SS2D_EINVAL;
    if (p->dstate > kTsMaxState || p->seqlen > INT32_MAX - 2 * kTsGrid) return SS2D_ENOTSUP;
    a.u = p->u; a.delta = p->delta; a.B = p->B; a.C = p->C; a.z = p->z; a.A = p->A; a.D = p->D; a.bias = p->delta_bias; a.initial = p->initial_state;
    a.cu = p->cu_seqlens; a.out = p->out; a.final = p->final_state; a.kept = p->kept_states;
    a.u_b = p->u_batch_stride; a.u_t = p->u_token_stride; a.dl_b = p->delta_batch_stride; a.dl_t = p->delta_token_stride; a.z_b = p->z_batch_stride; a.z_t = p->z_token_stride;
    a.B_b = p->B_batch_stride; a.B_t = p->B_token_stride; a.B_g = p->B_group_stride; a.C_b = p->C_batch_stride; a.C_t = p->C_token_stride; a.C_g = p->C_group_stride;
    a.batch = p->batch; a.tokens = p->seqlen; a.dim = p->dim; a.N = p->dstate; a.groups = p->n_groups; a.per_group = p->dim / p->n_groups;
    a.n_seqs = p->cu_seqlens ? p->n_seqs : p->batch; a.softplus = p->delta_softplus != 0;
    a.near = a.dim < 1 << 24;
    for (const int64_t stride : {a.u_t, a.dl_t, a.z_t, a.B_t, a.C_t}) a.near = a.near && stride >= 0 && stride < 1 << 24;
    a.keep = ts_keep(a.N);
    a.n_kept = (int)((a.tokens + (int64_t)a.keep - 1) / a.keep);
    if (a.dim) {
        if ((int64_t)a.dim * a.N > INT32_MAX - kBlock) return SS2D_ENOTSUP;
        ts_cut(a);
        const int64_t wgs = (int64_t)a.batch * a.n_segs * a.groups * a.wgs;
        if (wgs > kTsLaunch / kBlock || (int64_t)a.batch * a.n_segs > INT32_MAX || a.batch > 65535 * (a.n_segs > 1 ? 1 : 32768)) return SS2D_ENOTSUP;
    }
    return SS2D_OK;
}

// fn(T, sets, m) of the kernel that takes a state of N
template <typename T, typename F> static int ts_with(int N, F fn) {
    using std::integral_constant;
    if (N <= 4) return fn(T{}, integral_constant<int, 1>{}, integral_constant<int, 1>{});
    if (N <= 8) return fn(T{}, integral_constant<int, 2>{}, integral_constant<int, 1>{});
    if (N <= 16) return fn(T{}, integral_constant<int, 4>{}, integral_constant<int, 1>{});
    if (N <= 32) return fn(T{}, integral_constant<int, 4>{}, integral_constant<int, 2>{});
    return fn(T{}, integral_constant<int, 4>{}, integral_constant<int, 4>{});
}

// A state's tensors of sequences without tokens: the initial states, or zeros
__global__ __launch_bounds__(kBlock) void ts_copy_kernel(const float *from, float *to, int64_t n) {
    const int64_t i = (int64_t)blockIdx.x * kBlock + threadIdx.x;
    if (i < n) to[i] = from ? from[i] : 0.0f;
}
int ts_copy(const float *from, float *to, int64_t n, hipStream_t st) {
    if (!to || n == 0) return SS2D_OK;
    if ((n + kBlock - 1) / kBlock > kTsLaunch / kBlock) return SS2D_ENOTSUP;
    ts_copy_kernel<<<(uint32_t)((n + kBlock - 1) / kBlock), kBlock, 0, st>>>(from, to, n);
    return launch_status();
}

}  // namespace ss2d

using namespace ss2d;

extern "C" int64_t ss2d_token_scan_workspace_bytes(const ss2d_token_scan_params *params) {
    TsArgs a;
    const int rc = ts_read(params, a);
    if (rc != SS2D_OK) return rc;
    return a.dim && a.batch ? ts_carve(a, nullptr) : 0;
}

extern "C" int64_t ss2d_token_scan_kept_states(const ss2d_token_scan_params *params) {
    TsArgs a;
    const int rc = ts_read(params, a);
    if (rc == SS2D_OK && !ts_sums_fit(a)) return SS2D_ENOTSUP;       // (said by the forward that keeps states, not by the gradients at last)
    return rc != SS2D_OK ? rc : (int64_t)a.batch * a.n_kept * a.dim * a.N;
}

extern "C" int ss2d_token_scan_fwd(const ss2d_token_scan_params *params, void *workspace, int64_t workspace_bytes, void *stream) {
    TsArgs a;
    int rc = ts_read(params, a);
    if (rc != SS2D_OK || a.dim == 0 || a.batch == 0) return rc;
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    if (!a.A) return SS2D_EINVAL;
    if (a.tokens == 0) return ts_copy(a.initial, a.final, (int64_t)a.n_seqs * a.dim * a.N, st);
    if (!a.u || !a.delta || !a.B || !a.C || !a.out) return SS2D_EINVAL;
    const int64_t need = ts_carve(a, (uint8_t *)workspace);
    if (need && (!workspace || reinterpret_cast<uintptr_t>(workspace) % 16)) return SS2D_EINVAL;
    if (workspace_bytes < need) return SS2D_ENOMEM;
    auto run_as = [&](auto t, auto sets, auto m, auto quick) {
        using T = decltype(t);
        constexpr bool kQuick = decltype(quick)::value;
        const uint32_t wgs = (uint32_t)a.batch * a.groups * a.wgs;
        if (a.n_segs > 1) {
            ts_kernel<T, decltype(sets)::value, decltype(m)::value, true, kQuick><<<wgs * (a.n_segs - 1), kBlock, 0, st>>>(a);
            const uint32_t per_row = (uint32_t)a.dim * a.N;
            ts_join_kernel<<<dim3((per_row + kBlock - 1) / kBlock, a.batch), kBlock, 0, st>>>(a, per_row);
        }
        ts_kernel<T, decltype(sets)::value, decltype(m)::value, false, kQuick><<<wgs * a.n_segs, kBlock, 0, st>>>(a);
        return launch_status();
    };
    auto run = [&](auto t, auto sets, auto m) { return ts_quick(a) ? run_as(t, sets, m, std::true_type{}) : run_as(t, sets, m, std::false_type{}); };
    switch (params->dtype) {
    case SS2D_F32: return ts_with<float>(a.N, run);
    case SS2D_F16: return ts_with<f16_t>(a.N, run);
    default: return ts_with<bf16_t>(a.N, run);
    }
}
