// Gradients of linear attention with a decay for each head.  With E the gradient of the state behind a chunk, S the state before it,
// P_ts = scale exp(G_t - G_s) q_t . k_s and D_ts = scale exp(G_t - G_s) do_t . v_s for s <= t, 0 behind:
//     dq_t = sum_s D_ts k_s + scale exp(G_t) S do_t,     dk_s = sum_t D_ts q_t + exp(G_C - G_s) E v_s,
//     dv_s = sum_t P_ts do_t + exp(G_C - G_s) E^T k_s,   E before = exp(G_C) E + sum_t scale exp(G_t) q_t do_t^T.
// A decay g_t stands in every pair of a key before t and a query from t on, wherever the two are:
//     dg_t = sum_(s < t <= t') P_t's do_t' . v_s + sum_(t' >= t) scale exp(G_t') q_t' . (S do_t') + sum_(s < t) exp(G_C - G_s) k_s . (E v_s) + exp(G_C) <S, E>
// -- sums over the chunk alone.  (The shorter form, the sum of q . dq - k . dk from t to the sequence's end, is a small difference of
// long sums.)  S and E of all chunks come from two walks, and every chunk is then on its own.
#include <type_traits>

#include "linear_attention.h"

namespace ss2d {

// Sums over the lanes that hold the same column (four groups of 16), and over 16 columns
__device__ __forceinline__ float sum_groups(float v) { v += __shfl_xor(v, 16); return v + __shfl_xor(v, 32); }
__device__ __forceinline__ float sum_columns(float v) {
#pragma unroll
    for (int d = 1; d < 16; d *= 2) v += __shfl_xor(v, d);
    return v;
}

__device__ __forceinline__ float dot_frags(floatx4_t a, floatx4_t b) { return fmaf(a[0], b[0], a[1] * b[1]) + fmaf(a[2], b[2], a[3] * b[3]); }
__device__ __forceinline__ float dot_frags(u32x4_t a, u32x4_t b) {
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) sum = fmaf(unpack_lo<bf16_t>(a[i]), unpack_lo<bf16_t>(b[i]), fmaf(unpack_hi<bf16_t>(a[i]), unpack_hi<bf16_t>(b[i]), sum));
    return sum;
}
// Of states in three parts
__device__ __forceinline__ float dot_parts(u32x4_t a, const u32x4_t (&al)[2], u32x4_t b, const u32x4_t (&bl)[2]) {
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        sum = fmaf(unpack_lo<bf16_t>(a[i]) + (unpack_lo<bf16_t>(al[0][i]) + unpack_lo<bf16_t>(al[1][i])),
                   unpack_lo<bf16_t>(b[i]) + (unpack_lo<bf16_t>(bl[0][i]) + unpack_lo<bf16_t>(bl[1][i])), sum);
        sum = fmaf(unpack_hi<bf16_t>(a[i]) + (unpack_hi<bf16_t>(al[0][i]) + unpack_hi<bf16_t>(al[1][i])),
                   unpack_hi<bf16_t>(b[i]) + (unpack_hi<bf16_t>(bl[0][i]) + unpack_hi<bf16_t>(bl[1][i])), sum);
    }
    return sum;
}

// Eight wavefronts where a workgroup has a CU's LDS to itself, four where two or more share it
template <typename Op, int kDim> struct LaBwdShape {
    static constexpr bool kTile = sizeof(typename Op::E) == 2 && kDim <= kLaTurnDim;
    static constexpr int kC = Op::kChunk, kPitch = kDim + Op::kPad, kM = kC / 16;
    static constexpr int kTiles = (int)sizeof(typename Op::E) * (4 * kC * kPitch + 2 * kC * (kC + Op::kPad) + (kTile ? kDim * kPitch : 0));
    static constexpr int kWaves = kTiles > 78 * 1024 ? 8 : 4;
    static constexpr int kBytes = kTiles + (int)sizeof(float2) * kC + (int)sizeof(float) * (2 * kM * kC + 2 * kWaves * kC + kWaves + 1);
    static_assert(kBytes <= 160 * 1024, "LDS of a CU");
};

// A workgroup owns a chunk of one head: weights of its pairs to LDS, then its wavefronts take 16 columns of dq and dk, or of dv, at a time, as the
// outputs' kernel does (transposed products, states straight from memory; those of a wavefront's first columns are on their way from the start).
// kTile: E comes through LDS, where dk reads its rows and dv its columns; otherwise memory holds it both ways.
// kLow: dq's and dk's share of the states with what their rounding to bf16 left and what that one's left, for a decay's gradient in single precision.
// kDim: what both dimensions fit; the rows' pitch in LDS hangs on it, so that operands are read at fixed distances (170 -> 159 us below; where LDS then holds
// fewer workgroups it loses: keys of 48 with values of 80 in fp16 30 -> 35).
// 4 x 2048 tokens, 16 heads of 128 x 128, bf16: 158 us for 370 MB, 2.3 TB/s.  A workgroup has a CU's LDS to itself, so a chunk's loads (77 us of it) and its
// products take turns; a second chunk's rows in registers cost more in spills than they hid.
template <typename Op, typename T, int kDim, bool kLow, bool kFast>
__global__ __launch_bounds__((LaBwdShape<Op, kDim>::kWaves * kWave), 2) void la_bwd_kernel(const LaArgs p, float *head_sums, uint32_t total) {
    using E = typename Op::E;
    using Frag = typename Op::Frag;
    using Shape = LaBwdShape<Op, kDim>;
    constexpr bool kTile = Shape::kTile;
    constexpr int kWaves = Shape::kWaves, kPitch = Shape::kPitch, kPerRow = kDim / kVecOf<T>;
    constexpr int kC = Op::kChunk, kM = kC / 16, kVec = kVecOf<T>, kPitchP = kC + Op::kPad, kAhead = 4, kThreads = kWaves * kWave, kLower = kM * (kM + 1) / 2;
    extern __shared__ __align__(16) char lds[];
    const int dk = la_up(p.k.dim, Op::kStep), dv = la_up(p.v.dim, Op::kStep);
    E *qt = reinterpret_cast<E *>(lds), *kt = qt + kC * kPitch, *vt = kt + kC * kPitch, *ot = vt + kC * kPitch;
    E *pt = ot + kC * kPitch, *dt = pt + kC * kPitchP;              // P and D, as rows of a key's token
    const int sk = la_state_dim(p.k.dim), sv = la_state_dim(p.v.dim);
    E *et = dt + kC * kPitchP;
    float2 *cum = reinterpret_cast<float2 *>(et + (kTile ? kDim * kPitch : 0));
    float *of_queries = reinterpret_cast<float *>(cum + kC), *of_keys = of_queries + kM * kC;        // sums of the pairs' products, [16 keys / queries][token]
    float *with_s = of_keys + kM * kC, *with_e = with_s + kWaves * kC, *both = with_e + kWaves * kC;     // [wavefront][token], [wavefront]
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 15, quad = 4 * (lane >> 4);
    const uint32_t id = xcd_contiguous_id(blockIdx.x, total);
    const int c = id / (uint32_t)p.heads, h = id - (uint32_t)c * (uint32_t)p.heads;
    const int4 e = p.chunks[c];
    const int64_t entry = (int64_t)c * p.heads + h;
    if (e.z <= 0 || e.w < 0) {
        if (head_sums && tid == 0) head_sums[entry] = 0.0f;
        if (e.z <= 0) return;
    }
    const int64_t row0 = (int64_t)e.x * p.tokens + e.y;
    auto put = [&](const LaSide &side, int t, int d, floatx4_t v) {  // four values of a gradient, in single precision where heads are still to be summed
        const int64_t at = e.x * side.batch + (int64_t)(e.y + la_here(t)) * side.token + (int64_t)h * side.head + d;
        if (side.div > 1) store4(reinterpret_cast<float *>(side.p) + at, v, side.dim - d);
        else store4(reinterpret_cast<T *>(side.p) + at, v, side.dim - d);
    };
    auto put_decay = [&](int t, float v) {
        const int64_t at = (row0 + t) * p.heads + h;
        if (p.ddecay_f32) reinterpret_cast<float *>(p.ddecay)[at] = v;
        else reinterpret_cast<T *>(p.ddecay)[at] = from_f32<T>(v);
    };
    if (e.w < 0) {                                                   // rows of no sequence
        const floatx4_t none = {0, 0, 0, 0};
        for (int i = tid; i < e.z * (kLaMaxDim / 4); i += kThreads) {
            const int t = i / (kLaMaxDim / 4), d = i % (kLaMaxDim / 4) * 4;
            if (d < p.k.dim) { put(p.dq, t, d, none); put(p.dk, t, d, none); }
            if (d < p.v.dim) put(p.dv, t, d, none);
        }
        if (p.ddecay && !head_sums && tid < e.z) put_decay(tid, 0.0f);
        return;
    }
    // tasks of 16 columns: of dq and dk, then of dv
    const int key_tasks = (p.k.dim + 15) / 16, tasks = key_tasks + (p.v.dim + 15) / 16;
    const int4 seq = la_sequence(p, e.w);
    const bool has_s = e.y != seq.x || p.initial, has_e = e.y + e.z < seq.y || p.dfinal;
    const E *states = reinterpret_cast<const E *>(p.states) + entry * sk * sv, *dstates = reinterpret_cast<const E *>(p.dstates) + entry * sk * sv;
    const E *dstates_t = reinterpret_cast<const E *>(p.dstates_t) + entry * sk * sv;
    Frag s_ahead[kAhead], e_ahead[kAhead];                           // kAhead steps of a task's states
    auto fetch = [&](int task, int k0) {                             // (steps past the last repeat it, nobody uses them)
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            if (task < key_tasks) {
                const int at = min(k0 + k * Op::kStep, dv - Op::kStep);
                if (has_s) s_ahead[k] = Op::rows(states, sv, 16 * task, at, lane);
                if (!kTile && has_e) e_ahead[k] = Op::rows(dstates, sv, 16 * task, at, lane);
            } else if (!kTile && has_e) e_ahead[k] = Op::rows(dstates_t, sk, 16 * (task - key_tasks), min(k0 + k * Op::kStep, dk - Op::kStep), lane);
        }
    };

    {
        constexpr int kPieces = kC * kPerRow, kN = kPieces / kThreads < 1 ? 1 : kPieces / kThreads < 16 / kWaves ? kPieces / kThreads : 16 / kWaves;
        const LaSide *sides[4] = {&p.q, &p.k, &p.dout, &p.v};
        E *tiles[4] = {qt, kt, ot, vt};
        bool bad = false;
        if (tid < kC) cum[tid] = p.cum[entry * kC + tid];
        // (E is 16-bit and dense: kE pieces of 8 to a thread and pass)
        constexpr int kE = 4;
        const int e_row = sv / 8, e_pieces = sk * e_row;
        u32x4_t e_piece[kE];
        auto load_e = [&](int i) {
#pragma unroll
            for (int j = 0; j < kE; ++j) e_piece[j] = reinterpret_cast<const u32x4_t *>(dstates)[min(i + tid + j * kThreads, e_pieces - 1)];
        };
        auto put_e = [&](int i) {
#pragma unroll
            for (int j = 0; j < kE; ++j) {
                const int at = i + tid + j * kThreads, row = at / e_row;
                if (at < e_pieces) *reinterpret_cast<u32x4_t *>(et + row * kPitch + (at - row * e_row) * 8) = e_piece[j];
            }
        };
#pragma unroll
        for (int i = 0; i < kPieces; i += kN * kThreads) {
            u32x4_t piece[4][kN];
#pragma unroll
            for (int side = 0; side < 4; ++side) {
                const LaSide &from = *sides[side];
                const T *src = reinterpret_cast<const T *>(from.p) + e.x * from.batch + (int64_t)e.y * from.token + (int64_t)(h / from.div) * from.head;
#pragma unroll
                for (int j = 0; j < kN; ++j) {
                    const int at = i + tid + j * kThreads;
                    piece[side][j] = load_piece<kFast>(src, from.token, at / kPerRow, e.z, at % kPerRow * kVec, from.dim);
                }
            }
            if (i == 0) {
                if (kTile && has_e) load_e(0);
                if (wave < tasks) fetch(wave, 0);
            }
#pragma unroll
            for (int side = 0; side < 4; ++side)
#pragma unroll
                for (int j = 0; j < kN; ++j) {
                    const int at = i + tid + j * kThreads, r = at / kPerRow, d = at % kPerRow * kVec;
                    if (kPieces % (kN * kThreads) == 0 || r < kC) {
                        const u32x4_t held = held_piece<kFast, T>(piece[side][j], r < e.z, d, sides[side]->dim);
                        put_piece<T, E>(tiles[side] + r * kPitch + d, held);
                        if (side < 3) bad |= piece_bad<T>(held);
                    }
                }
        }
        if (kTile && has_e) {
            put_e(0);
            for (int i = kE * kThreads; i < e_pieces; i += kE * kThreads) {
                load_e(i);
                put_e(i);
            }
        }
        if (tid == 0) both[kWaves] = 0.0f;
        __syncthreads();
        if (bad) both[kWaves] = 1.0f;
    }

    // weights of the pairs: tiles of 16 x 16 below and on the diagonal first, then zeros
    for (int k = wave; k < kM * kM; k += kWaves) {
        int tt = k < 1 ? 0 : k < 3 ? 1 : k < 6 ? 2 : 3, ts = k - tt * (tt + 1) / 2;
        if (k >= kLower) {
            const int u = k - kLower;
            ts = u < 1 ? 1 : u < 3 ? 2 : 3;
            tt = u - ts * (ts - 1) / 2;
        }
        floatx4_t weights = {0, 0, 0, 0}, through = {0, 0, 0, 0}, product = {0, 0, 0, 0};
        const int t = 16 * tt + quad, s = 16 * ts + col;
        if (ts <= tt) {
            for (int k0 = 0; k0 < dk; k0 += Op::kStep)
                weights = Op::mma(Op::rows(qt, kPitch, 16 * tt, k0, lane), Op::rows(kt, kPitch, 16 * ts, k0, lane), weights);
            for (int k0 = 0; k0 < dv; k0 += Op::kStep)
                through = Op::mma(Op::rows(ot, kPitch, 16 * tt, k0, lane), Op::rows(vt, kPitch, 16 * ts, k0, lane), through);
            const float2 gs = cum[s];
#pragma unroll
            for (int v = 0; v < 4; ++v) {
                const float2 gt = cum[t + v];
                const float decay = fast_exp2((gt.x - gs.x) + (gt.y - gs.y)) * p.scale, weight = weights[v] * decay, pair = weight * through[v],
                            back = through[v] * decay;
                weights[v] = s <= t + v ? weight : 0.0f;
                product[v] = s < t + v ? pair : 0.0f;                // (a pair of one token has no decay between)
                through[v] = s <= t + v ? back : 0.0f;
            }
        }
        Op::put4_places(pt + s * kPitchP, t, weights);
        Op::put4(dt + s * kPitchP + t, through);
        if (!p.ddecay) continue;
        // of these 16 x 16 pairs: sums for each query and each key; on the diagonal, for each token the pairs that it stands between
        const float of_key = sum_groups((product[0] + product[1]) + (product[2] + product[3]));
        if (lane < 16) of_keys[tt * kC + s] = ts < tt ? of_key : 0.0f;
        if (ts == tt) {
            product[2] += product[3];                                // from a query on
            product[1] += product[2];
            product[0] += product[1];
            const float next = __shfl_down(product[0], 16), third = __shfl_down(product[0], 32), fourth = __shfl_down(product[0], 48);
            const float behind = (lane < 48 ? next : 0.0f) + (lane < 32 ? third : 0.0f) + (lane < 16 ? fourth : 0.0f);
#pragma unroll
            for (int v = 0; v < 4; ++v) product[v] = col < quad + v ? product[v] + behind : 0.0f;
        }
#pragma unroll
        for (int v = 0; v < 4; ++v) {
            const float of_query = sum_columns(product[v]);
            if (col == 0) of_queries[ts * kC + t + v] = of_query;
        }
    }
    __syncthreads();

    const bool bad = both[kWaves] != 0.0f;
    const float2 end = cum[kC - 1];
    float q_dot[kM], k_dot[kM], se = 0.0f, in[kM], out[kM];          // of a token: the decay from what came in, to what goes out
#pragma unroll
    for (int m = 0; m < kM; ++m) {
        const float2 g = cum[16 * m + col];
        q_dot[m] = k_dot[m] = 0.0f;
        in[m] = p.scale * fast_exp2(g.x + g.y);
        out[m] = fast_exp2((end.x - g.x) + (end.y - g.y));
    }
    for (int task = wave; task < tasks; task += kWaves) {
        if (task < key_tasks) {
            const int n = task;
            floatx4_t dq[kM], dkey[kM];
#pragma unroll
            for (int m = 0; m < kM; ++m) dq[m] = dkey[m] = floatx4_t{0, 0, 0, 0};
            for (int g = 0; g < dv && (has_s || has_e); g += kAhead * Op::kStep) {
                if (g) fetch(task, g);                               // (the first ones: from the start, or from the task before)
#pragma unroll
                for (int k = 0; k < kAhead; ++k) {
                    const int k0 = g + k * Op::kStep;
                    if (k0 >= dv) break;
                    if (kTile && has_e) e_ahead[k] = Op::rows(et, kPitch, 16 * n, k0, lane);
                    Frag sl[2], dl[2];
                    if constexpr (kLow)
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            if (has_s) sl[i] = Op::rows(states + (1 + i) * p.low, sv, 16 * n, k0, lane);
                            if (has_e) dl[i] = Op::rows(dstates + (1 + i) * p.low, sv, 16 * n, k0, lane);
                        }
                    if (has_s)
#pragma unroll
                        for (int m = 0; m < kM; ++m) {
                            const Frag o = Op::rows(ot, kPitch, 16 * m, k0, lane);
                            dq[m] = Op::mma(s_ahead[k], o, dq[m]);
                            if constexpr (kLow)
#pragma unroll
                                for (int i = 0; i < 2; ++i) dq[m] = Op::mma(sl[i], o, dq[m]);
                        }
                    if (has_e)
#pragma unroll
                        for (int m = 0; m < kM; ++m) {
                            const Frag v = Op::rows(vt, kPitch, 16 * m, k0, lane);
                            dkey[m] = Op::mma(e_ahead[k], v, dkey[m]);
                            if constexpr (kLow)
#pragma unroll
                                for (int i = 0; i < 2; ++i) dkey[m] = Op::mma(dl[i], v, dkey[m]);
                        }
                    if (has_s && has_e && p.ddecay) {
                        if constexpr (kLow) se += dot_parts(s_ahead[k], sl, e_ahead[k], dl);
                        else se += dot_frags(s_ahead[k], e_ahead[k]);
                    }
                }
            }
            if (task + kWaves < tasks) fetch(task + kWaves, 0);
#pragma unroll
            for (int m = 0; m < kM; ++m) {
                const E *q = qt + (16 * m + col) * kPitch + 16 * n + quad, *k = kt + (16 * m + col) * kPitch + 16 * n + quad;
                dq[m] *= in[m];
                dkey[m] *= out[m];
#pragma unroll
                for (int v = 0; v < 4; ++v) {
                    q_dot[m] = fmaf(dq[m][v], to_f32(q[v]), q_dot[m]);
                    k_dot[m] = fmaf(dkey[m][v], to_f32(k[v]), k_dot[m]);
                }
            }
            if (!bad) {
#pragma unroll
                for (int k0 = 0; k0 < kC; k0 += Op::kStep) {
                    const Frag k = Op::cols(kt, kPitch, 16 * n, k0, lane), q = Op::cols(qt, kPitch, 16 * n, k0, lane);
#pragma unroll
                    for (int m = 0; m < kM; ++m) {
                        if (16 * m >= k0) dq[m] = Op::mma(k, Op::cols(dt, kPitchP, 16 * m, k0, lane), dq[m]);
                        if (16 * m < k0 + Op::kStep) dkey[m] = Op::mma(q, Op::in_places(Op::rows(dt, kPitchP, 16 * m, k0, lane)), dkey[m]);
                    }
                }
            } else {                                                 // as in the outputs' kernel: nothing from behind the diagonal
                const int c0 = la_here(col), d0 = la_here(16 * n + quad);
#pragma unroll
                for (int m = 0; m < kM; ++m) {
                    const int own = 16 * m + c0;
                    for (int r = 0; r < kC; ++r)
#pragma unroll
                        for (int v = 0; v < 4; ++v) {
                            if (r <= own) dq[m][v] += to_f32(dt[r * kPitchP + own]) * to_f32(kt[r * kPitch + d0 + v]);
                            if (r >= own) dkey[m][v] += to_f32(dt[own * kPitchP + r]) * to_f32(qt[r * kPitch + d0 + v]);
                        }
                }
            }
#pragma unroll
            for (int m = 0; m < kM; ++m)
                if (16 * m + col < e.z) {
                    put(p.dq, 16 * m + col, 16 * n + quad, dq[m]);
                    put(p.dk, 16 * m + col, 16 * n + quad, dkey[m]);
                }
        } else {
            const int n = task - key_tasks;
            floatx4_t acc[kM];
#pragma unroll
            for (int m = 0; m < kM; ++m) acc[m] = floatx4_t{0, 0, 0, 0};
            if (kTile && has_e) {
                for (int k0 = 0; k0 < dk; k0 += Op::kStep) {
                    const Frag a = Op::cols(et, kPitch, 16 * n, k0, lane);
#pragma unroll
                    for (int m = 0; m < kM; ++m) acc[m] = Op::mma(a, Op::in_places(Op::rows(kt, kPitch, 16 * m, k0, lane)), acc[m]);
                }
            }
            for (int g = 0; !kTile && g < dk && has_e; g += kAhead * Op::kStep) {
                if (g || (task != wave && task - kWaves >= key_tasks)) fetch(task, g);
#pragma unroll
                for (int k = 0; k < kAhead; ++k) {
                    if (g + k * Op::kStep >= dk) break;
#pragma unroll
                    for (int m = 0; m < kM; ++m) acc[m] = Op::mma(e_ahead[k], Op::rows(kt, kPitch, 16 * m, g + k * Op::kStep, lane), acc[m]);
                }
            }
#pragma unroll
            for (int m = 0; m < kM; ++m) acc[m] *= out[m];
            if (!bad) {
#pragma unroll
                for (int k0 = 0; k0 < kC; k0 += Op::kStep) {
                    const Frag o = Op::cols(ot, kPitch, 16 * n, k0, lane);
#pragma unroll
                    for (int m = 0; m < kM; ++m)
                        if (16 * m < k0 + Op::kStep) acc[m] = Op::mma(o, Op::rows(pt, kPitchP, 16 * m, k0, lane), acc[m]);
                }
            } else {
                const int c0 = la_here(col), d0 = la_here(16 * n + quad);
#pragma unroll
                for (int m = 0; m < kM; ++m)
                    for (int r = 16 * m + c0; r < kC; ++r)
#pragma unroll
                        for (int v = 0; v < 4; ++v) acc[m][v] += to_f32(pt[(16 * m + c0) * kPitchP + Op::place(r)]) * to_f32(ot[r * kPitch + d0 + v]);
            }
#pragma unroll
            for (int m = 0; m < kM; ++m)
                if (16 * m + col < e.z) put(p.dv, 16 * m + col, 16 * n + quad, acc[m]);
        }
    }
    if (!p.ddecay) return;

#pragma unroll
    for (int m = 0; m < kM; ++m) {
        const float a = sum_groups(q_dot[m]), b = sum_groups(k_dot[m]);
        if (lane < 16) {
            with_s[wave * kC + 16 * m + col] = a;
            with_e[wave * kC + 16 * m + col] = b;
        }
    }
    se = sum_groups(sum_columns(se));
    if (lane == 0) both[wave] = se;
    __syncthreads();
    if (wave != 0) return;
    // The pairs that a token t stands between: of its own 16 tokens, of those with earlier keys (from t on), of those with later queries (before t), of
    // earlier keys and later queries; then those of what came in (from t on) and of what goes out (before t).
    float between = 0.0f, from = 0.0f, until = 0.0f, after = 0.0f, before = 0.0f, states_both = 0.0f;
    const int own = lane / 16;
    if (lane < kC) {
        between = of_queries[own * kC + lane];
        for (int i = 0; i < own; ++i) from += of_queries[i * kC + lane];
        for (int i = own + 1; i < kM; ++i) until += of_keys[i * kC + lane];
#pragma unroll
        for (int i = 0; i < kWaves; ++i) {
            after += with_s[i * kC + lane];
            before += with_e[i * kC + lane];
        }
    }
#pragma unroll
    for (int i = 0; i < kWaves; ++i) states_both += both[i];
#pragma unroll
    for (int m = 1; m + 1 < kM; ++m) {
        float over = 0.0f;
        if (own < m)
            for (int i = m + 1; i < kM; ++i) over += of_keys[i * kC + lane];
        over = sum_groups(sum_columns(over));
        if (own == m) between += over;
    }
#pragma unroll
    for (int d = 1; d < 16; d *= 2) {
        const float a = __shfl_down(from, d), b = __shfl_up(until, d);
        if (col + d < 16) from += a;
        if (col >= d) until += b;
    }
#pragma unroll
    for (int d = 1; d < kC; d *= 2) {
        const float a = __shfl_down(after, d), b = __shfl_up(before, d);
        if (lane + d < kC) after += a;
        if (lane >= d) before += b;
    }
    const float until_t = __shfl_up(until, 1), before_t = __shfl_up(before, 1);      // (a token's key is not before it)
    LaKeep<E> keep;
    keep.set(end, p.kept + entry);
    float dg = between + from + (col > 0 ? until_t : 0.0f) + after + (lane > 0 ? before_t : 0.0f) + keep.of(states_both);
    if (head_sums) {
        dg = sum_groups(sum_columns(lane < e.z ? dg : 0.0f));
        if (lane == 0) head_sums[entry] = dg;
    } else if (lane < e.z) put_decay(lane, dg);
}

// Gradients of what several heads share: the heads' sum, of `per` neighbouring values in single precision, dim apart
// (dimensions that four divides: four neighbours to a thread).
struct LaSum {
    const float *x;
    void *out;
    int64_t total;                   // results, in units of kVec
    int32_t dim, per;                // of a head, in units of kVec; heads to one
};
struct LaSums { LaSum side[3]; };
template <typename T, int kVec> __global__ __launch_bounds__(kBlock) void la_sum_heads_kernel(const LaSums sums) {
    int64_t i = (int64_t)blockIdx.x * kBlock + threadIdx.x;
    LaSum s = sums.side[0];
#pragma unroll
    for (int k = 1; k < 3; ++k)
        if (i >= s.total) {
            i -= s.total;
            s = sums.side[k];
        }
    if (i >= s.total) return;
    const int64_t group = i / s.dim, at = group * s.per * s.dim + (i - group * s.dim);
    float sum[kVec];
#pragma unroll
    for (int v = 0; v < kVec; ++v) sum[v] = 0.0f;
    if constexpr (kVec == 4) {
        const floatx4_t *x = reinterpret_cast<const floatx4_t *>(s.x) + at;
#pragma unroll 4
        for (int k = 0; k < s.per; ++k) {
            const floatx4_t more = x[(int64_t)k * s.dim];
#pragma unroll
            for (int v = 0; v < 4; ++v) sum[v] += more[v];
        }
        store4(reinterpret_cast<T *>(s.out) + 4 * i, floatx4_t{sum[0], sum[1], sum[2], sum[3]}, 4);
    } else {
#pragma unroll 4
        for (int k = 0; k < s.per; ++k) sum[0] += s.x[at + (int64_t)k * s.dim];
        reinterpret_cast<T *>(s.out)[i] = from_f32<T>(sum[0]);
    }
}

// A learnt decay's gradient: the chunks' sums of its head, a workgroup to a head
template <typename T> __global__ __launch_bounds__(kBlock) void la_sum_decays_kernel(const float *sums, void *out, int chunks, int heads, int f32) {
    __shared__ double part[kBlock];
    const int h = blockIdx.x, tid = threadIdx.x;
    double sum = 0.0;
    for (int c = tid; c < chunks; c += kBlock) sum += (double)sums[(int64_t)c * heads + h];
    part[tid] = sum;
    for (int d = kBlock / 2; d >= 1; d /= 2) {
        __syncthreads();
        if (tid < d) part[tid] += part[tid + d];
    }
    if (tid != 0) return;
    if (f32) reinterpret_cast<float *>(out)[h] = (float)part[0];
    else reinterpret_cast<T *>(out)[h] = from_f32<T>((float)part[0]);
}

struct LaBackward {
    LaArgs a;
    bool low;
    float *head_sums;
    void *dq, *dk, *dv;              // where the heads' sums go
};

template <typename Op, typename T> static int la_backward(const LaBackward &b, float *dinitial, void *stream) {
    const LaArgs &p = b.a;
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    int rc = la_tables(p, Op::kChunk, 0, stream);
    if (rc != SS2D_OK) return rc;
    // S by keys, dense along values; E the same way, and for dv by values, dense along keys
    LaWalk w[2] = {};
    int n = 0;
    const bool one = !p.cu && p.per_seq <= 1;                        // a chunk to a sequence: nothing comes in but what the caller gives
    if (!one || p.initial) {
        LaWalk &s = w[n];
        s.a = p.v; s.b = p.k;
        s.out = p.states; s.low = p.low;
        s.from = p.initial;
        s.local = p.local + n++ * p.local_floats;
    }
    if (!one || p.dfinal || dinitial) {
        LaWalk &s = w[n];
        s.a = p.dout; s.b = p.q;
        s.out = p.dstates; s.out_t = la_turned(p, sizeof(typename Op::E) == 2 ? SS2D_BF16 : SS2D_F32) ? p.dstates_t : nullptr; s.low = p.low;
        s.from = p.dfinal; s.to = dinitial;
        s.reverse = 1;
        s.exact = dinitial != nullptr;
        s.local = p.local + n++ * p.local_floats;
    }
    for (LaWalk &s : w) {
        s.from_a = 1; s.from_b = p.v.dim;
        s.exact = s.exact || p.low != 0;
    }
    if (n && (rc = la_walks<Op, T>(p, w, n, stream)) != SS2D_OK) return rc;
    const uint32_t total = (uint32_t)p.max_chunks * (uint32_t)p.heads;
    if (total > 0) {
        const bool fast = p.q.pieces && p.k.pieces && p.v.pieces && p.dout.pieces;
        auto go = [&](auto kernel, int waves, int bytes) {
            // (up to 157 KB of LDS: this runtime asks for no attribute above 64)
            kernel<<<total, waves * kWave, bytes, st>>>(p, b.head_sums, total);
            return launch_status();
        };
        auto sized = [&](auto dim) {
            constexpr int kDim = decltype(dim)::value, kWaves = LaBwdShape<Op, kDim>::kWaves, kBytes = LaBwdShape<Op, kDim>::kBytes;
            constexpr bool k16 = sizeof(typename Op::E) == 2;
            if (k16 && b.low) return fast ? go(la_bwd_kernel<Op, T, kDim, k16, true>, kWaves, kBytes) : go(la_bwd_kernel<Op, T, kDim, k16, false>, kWaves, kBytes);
            return fast ? go(la_bwd_kernel<Op, T, kDim, false, true>, kWaves, kBytes) : go(la_bwd_kernel<Op, T, kDim, false, false>, kWaves, kBytes);
        };
        const int dim = p.k.dim > p.v.dim ? p.k.dim : p.v.dim;
        rc = dim <= 64 ? sized(std::integral_constant<int, 64>{}) : dim <= 128 ? sized(std::integral_constant<int, 128>{}) : sized(std::integral_constant<int, 256>{});
        if (rc != SS2D_OK) return rc;
        LaSums sums = {};
        int n_sums = 0;
        int64_t values = 0;
        bool fours = true;
        auto sum = [&](const LaSide &side, void *out) {
            if (side.div <= 1) return;
            const int64_t heads = (int64_t)p.batch * p.tokens * (p.heads / side.div);
            sums.side[n_sums++] = LaSum{reinterpret_cast<const float *>(side.p), out, heads * side.dim, side.dim, side.div};
            values += heads * side.dim;
            fours = fours && side.dim % 4 == 0;
        };
        sum(p.dq, b.dq);
        sum(p.dk, b.dk);
        sum(p.dv, b.dv);
        if (fours)
            for (LaSum &s : sums.side) { s.total /= 4; s.dim /= 4; }
        const int64_t each = fours ? kBlock * 4 : kBlock;
        if (values > 0 && fours) la_sum_heads_kernel<T, 4><<<(uint32_t)((values + each - 1) / each), kBlock, 0, st>>>(sums);
        else if (values > 0) la_sum_heads_kernel<T, 1><<<(uint32_t)((values + each - 1) / each), kBlock, 0, st>>>(sums);
    }
    if (b.head_sums) la_sum_decays_kernel<T><<<p.heads, kBlock, 0, st>>>(b.head_sums, p.ddecay, p.max_chunks, p.heads, p.ddecay_f32);
    return launch_status();
}

LaSide la_side(const void *ptr, int64_t batch, int64_t token, int64_t head, int heads, int own_heads, int dim, int size);
int la_arguments(const ss2d_linear_attention_params *p, LaArgs &a, bool &empty);
int la_chunk(int dtype);
int64_t la_carve(LaArgs &p, int dtype, char *base, bool backward, bool low);

// Everything of a backward call, its workspace laid out from `base` on; the bytes that takes, or a status.
static int64_t la_backward_plan(const ss2d_linear_attention_bwd_params *params, LaBackward &b, bool &empty, char *base) {
    empty = false;
    if (!params) return SS2D_EINVAL;
    const ss2d_linear_attention_params &f = params->fwd;
    const int rc = la_arguments(&f, b.a, empty);
    if (rc != SS2D_OK || empty) return rc;
    LaArgs &a = b.a;
    const int planned = la_plan(a, la_chunk(f.dtype), (int64_t)((f.key_dim + kLaTile - 1) / kLaTile) * ((f.value_dim + kLaTile - 1) / kLaTile) * 2, 4, kLaThreads);
    if (planned != SS2D_OK) return planned;
    const int size = f.dtype == SS2D_F32 ? 4 : 2;
    if (params->ddecay && !f.decay) return SS2D_EINVAL;
    b.low = f.dtype == SS2D_BF16 && params->ddecay && f.decay_dtype == SS2D_F32;
    a.dout = la_side(params->dout, params->dout_batch_stride, params->dout_token_stride, params->dout_head_stride, f.heads, f.heads, f.value_dim, size);
    a.dfinal = params->dfinal_state;
    a.ddecay = params->ddecay;
    a.ddecay_f32 = f.decay_dtype == SS2D_F32;
    int64_t at = la_carve(a, f.dtype, base, true, b.low);
    auto gradient = [&](LaSide &side, void *&to, void *ptr, int own, int dim) {
        const bool shared = own != f.heads;
        to = ptr;
        const int64_t row = (int64_t)f.heads * dim;
        side = la_side(shared ? base + at : ptr, row * f.seqlen, row, dim, f.heads, own, dim, shared ? 4 : size);
        if (shared) at += (4 * row * f.seqlen * f.batch + 255) / 256 * 256;
    };
    gradient(a.dq, b.dq, params->dq, f.q_heads, f.key_dim);
    gradient(a.dk, b.dk, params->dk, f.k_heads, f.key_dim);
    gradient(a.dv, b.dv, params->dv, f.v_heads, f.value_dim);
    b.head_sums = nullptr;
    if (params->ddecay && params->decay_per_head) {
        b.head_sums = reinterpret_cast<float *>(base + at);
        at += ((int64_t)4 * a.max_chunks * a.heads + 255) / 256 * 256;
    }
    return at;
}

// No sequence at all: what all tokens of a head share has a gradient still, the sum of none
static int la_no_decays(const ss2d_linear_attention_bwd_params &g, hipStream_t st) {
    const ss2d_linear_attention_params &f = g.fwd;
    if (!g.ddecay || !g.decay_per_head || f.heads == 0) return SS2D_OK;
    if (!f.decay) return SS2D_EINVAL;
    if (f.decay_dtype == SS2D_F16) la_sum_decays_kernel<f16_t><<<f.heads, kBlock, 0, st>>>(nullptr, g.ddecay, 0, f.heads, 0);
    else la_sum_decays_kernel<bf16_t><<<f.heads, kBlock, 0, st>>>(nullptr, g.ddecay, 0, f.heads, f.decay_dtype == SS2D_F32);
    return launch_status();
}

}  // namespace ss2d

using namespace ss2d;

extern "C" int64_t ss2d_linear_attention_bwd_workspace_bytes(const ss2d_linear_attention_bwd_params *params) {
    LaBackward b;
    bool empty;
    return la_backward_plan(params, b, empty, nullptr);
}

extern "C" int ss2d_linear_attention_bwd(const ss2d_linear_attention_bwd_params *params, void *workspace, int64_t workspace_bytes, void *stream) {
    LaBackward b;
    bool empty;
    const int64_t need = la_backward_plan(params, b, empty, reinterpret_cast<char *>(workspace));
    if (need < 0) return (int)need;
    if (empty) return la_no_decays(*params, reinterpret_cast<hipStream_t>(stream));
    if (b.a.tokens > 0 && (!params->dout || !params->dq || !params->dk || !params->dv)) return SS2D_EINVAL;
    if (!workspace || (uintptr_t)workspace % 16 != 0) return SS2D_EINVAL;
    if (workspace_bytes < need) return SS2D_ENOMEM;
    switch (params->fwd.dtype) {
    case SS2D_F32: return la_backward<OperandF32, float>(b, params->dinitial_state, stream);
    case SS2D_F16: return la_backward<OperandF32, f16_t>(b, params->dinitial_state, stream);
    default: return la_backward<OperandBf16, bf16_t>(b, params->dinitial_state, stream);
    }
}
