// Norm and position rotation of the queries and keys of an attention, one pass for both: a row is one head of one token,
//     n = x rsqrt(mean(x^2) + eps) w,   (a, b) -> (a cos - b sin, b cos + a sin) for the pairs of the first R values of n,
// the angle of pair i = axis * F + f the token's position on that axis times frequency (axis, f).  Its gradient, with d = dy turned back:
//     dw = sum over the rows of d xhat,   dx = r (w d - xhat mean(w d xhat)),   xhat = x r,   r = rsqrt(mean(x^2) + eps) computed again.
// Memory bounds both: every value is read and written once.  A row lives in the registers of 4 to 64 lanes, 8 values each -- of half-split
// pairs four first and four second values, so that no pair spans two lanes -- and the weights stay there too.  Angles are computed
// once per token and pair for all its heads, in LDS: a product in 64 bits, its whole turns taken off there (a position of a million
// times a frequency has no digits left for the fraction in 32), and then sine and cosine in single precision.
// 4 x 4096 tokens of 32 + 8 heads of 128, bf16: 66 us for 335 MB, 5.1 TB/s, what a copy reaches; backward 116 for 503 MB, 4.3 TB/s (two rows of a lane in
// flight instead of four, for its registers).  Rounds of one token took 153 us each: 40 rows leave most lanes of the last step idle.
#include "ss2d_common.h"

namespace ss2d {

constexpr int kQnMaxDim = 512;       // 64 lanes x 8
constexpr int kQnTokens = 16;        // of one round of a workgroup, at most
constexpr int kQnPairs = 1024;       // angles in LDS

struct QnSide {
    const void *x, *dy;              // (batch, token, head, dim) by strides, the last dimension dense
    void *y;                         // dense; forward: the result, backward: dx
    const void *w;                   // (dim) or NULL
    int64_t batch, token, head, dy_batch, dy_token, dy_head;
    int32_t heads;
};

struct QnArgs {
    QnSide side[2];
    const void *positions;           // (batch, token, axis) by strides, or NULL: no rotation
    const void *frequencies;         // (axes, per_axis), dense
    int64_t pos_batch, pos_token, pos_axis;
    int32_t pos64, freq64, axes, per_axis, pairs;                    // pairs = axes * per_axis
    int32_t batch, tokens, dim, w_dtype, interleaved, round, has_w;  // round: tokens of a workgroup's round
    int64_t rounds;
    FastDiv by_heads[2], by_pairs, by_tokens;
    float eps;
    float *partial;                  // backward: [workgroup][side][dim]
};

__device__ __forceinline__ float qn_weight(const void *w, int at, int dtype) {
    return !w ? 1.0f : dtype == SS2D_F32 ? reinterpret_cast<const float *>(w)[at]
                     : dtype == SS2D_BF16 ? to_f32(reinterpret_cast<const bf16_t *>(w)[at]) : to_f32(reinterpret_cast<const f16_t *>(w)[at]);
}

// (cos, sin) of one pair of a token.  For results in 16 bits the hardware's sine and cosine of a part of a turn do: off by 1.3e-7 at most.
template <typename T> __device__ __forceinline__ float2 qn_angle(const QnArgs &p, int b, int t, int pair) {
    const int axis = p.axes == 1 ? 0 : pair / p.per_axis;
    const int64_t at = b * p.pos_batch + t * p.pos_token + axis * p.pos_axis;
    const double pos = p.pos64 ? (double)reinterpret_cast<const int64_t *>(p.positions)[at] : (double)reinterpret_cast<const int32_t *>(p.positions)[at];
    const double f = p.freq64 ? reinterpret_cast<const double *>(p.frequencies)[pair] : (double)reinterpret_cast<const float *>(p.frequencies)[pair];
    const double turns = pos * f * 0.15915494309189535;              // 1 / (2 pi)
    const float part = (float)(turns - rint(turns));
    if constexpr (sizeof(T) == 2) return make_float2(__builtin_amdgcn_cosf(part), __builtin_amdgcn_sinf(part));
    float s, c;
    sincospif(2.0f * part, &s, &c);
    return make_float2(c, s);
}

// The lane's 8 values: two fours, which of half-split pairs are the pairs' first and second values
template <typename T> __device__ __forceinline__ void qn_load4(const T *p, float *v) {
    if constexpr (sizeof(T) == 4) {
        const floatx4_t q = *reinterpret_cast<const floatx4_t *>(p);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = q[i];
    } else {
        const uint2 q = *reinterpret_cast<const uint2 *>(p);
        v[0] = unpack_lo<T>(q.x); v[1] = unpack_hi<T>(q.x); v[2] = unpack_lo<T>(q.y); v[3] = unpack_hi<T>(q.y);
    }
}
template <typename T> __device__ __forceinline__ void qn_store4(T *p, const float *v) {
    if constexpr (sizeof(T) == 4) *reinterpret_cast<floatx4_t *>(p) = floatx4_t{v[0], v[1], v[2], v[3]};
    else *reinterpret_cast<uint2 *>(p) = make_uint2(pack2_from_f32<T>(v[0], v[1]), pack2_from_f32<T>(v[2], v[3]));
}

// One pair turned, forward or back
__device__ __forceinline__ void qn_turn(float &a, float &b, float2 cs, bool back) {
    const float s = back ? -cs.y : cs.y, x = a;
    a = x * cs.x - b * s;
    b = b * cs.x + x * s;
}
__device__ __forceinline__ void qn_turn8(float (&v)[8], const float2 *cs, bool interleaved, bool back) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 c = cs[i];
        if (interleaved) qn_turn(v[2 * i], v[2 * i + 1], c, back);
        else qn_turn(v[i], v[4 + i], c, back);
    }
}

// Sum over the kLanes lanes of a row, in each of them: neighbours, pairs, the other four, the other eight by lane moves inside the addition
template <int kLanes> __device__ __forceinline__ float qn_sum(float v) {
    v += dpp_move<0xB1>(0.0f, v);
    v += dpp_move<0x4E>(0.0f, v);
    if constexpr (kLanes >= 8) v += dpp_move<0x141>(0.0f, v);
    if constexpr (kLanes >= 16) v += dpp_move<0x140>(0.0f, v);
    if constexpr (kLanes >= 32) v += __shfl_xor(v, 16);
    if constexpr (kLanes >= 64) v += __shfl_xor(v, 32);
    return v;
}

// kLanes lanes to a row.  A workgroup takes rounds of p.round tokens: their angles and places, then all heads of queries, then of keys.
template <typename T, int kLanes, bool kBack>
__global__ __launch_bounds__(kBlock) void qk_norm_rotate_kernel(const QnArgs p) {
    constexpr int kSlots = kBlock / kLanes, kAhead = kBack ? 2 : 4;
    __shared__ float2 angles[kQnPairs];
    __shared__ int64_t places[4][kQnTokens];                         // of a token's first head: x of queries and of keys, dy of both
    __shared__ float sums[kBack ? kBlock * 8 : 1];
    const int tid = threadIdx.x, slot = tid / kLanes, unit = tid % kLanes;
    const bool in = 8 * unit < p.dim, turned = 4 * unit < p.pairs && p.positions;
    const int first = !in ? 0 : turned && !p.interleaved ? 4 * unit : 8 * unit, second = !in ? 4 : turned && !p.interleaved ? p.pairs + 4 * unit : 8 * unit + 4;
    const float inv_d = 1.0f / (float)p.dim;
    const int64_t all = (int64_t)p.batch * p.tokens;
    float w[2][8], dw[2][8];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            w[k][i] = 1.0f;
            dw[k][i] = 0.0f;
        }
        if (!p.side[k].w) continue;                                  // (T's own type otherwise; all four loads are on their way at once)
        if (p.w_dtype == SS2D_F32) {
            qn_load4(reinterpret_cast<const float *>(p.side[k].w) + first, w[k]);
            qn_load4(reinterpret_cast<const float *>(p.side[k].w) + second, w[k] + 4);
        } else {
            qn_load4(reinterpret_cast<const T *>(p.side[k].w) + first, w[k]);
            qn_load4(reinterpret_cast<const T *>(p.side[k].w) + second, w[k] + 4);
        }
    }
    for (int64_t round = blockIdx.x; round < p.rounds; round += gridDim.x) {
        const int64_t token0 = round * p.round;
        const int n_tokens = (int)(all - token0 < p.round ? all - token0 : p.round);
        uint32_t b0, t0;
        if (all <= 0x7fffffff) divmod((uint32_t)token0, p.by_tokens, b0, t0);
        else { b0 = (uint32_t)(token0 / p.tokens); t0 = (uint32_t)(token0 - (int64_t)b0 * p.tokens); }
        auto place = [&](int t, int &b, int &at) {                   // the round's t-th token
            b = (int)b0;
            at = (int)t0 + t;
            while (at >= p.tokens) { at -= p.tokens; ++b; }
        };
        if (round != blockIdx.x) __syncthreads();
        if (tid < 4 * kQnTokens && tid % kQnTokens < n_tokens) {
            const int what = tid / kQnTokens;
            const QnSide &s = p.side[what % 2];
            int b, at;
            place(tid % kQnTokens, b, at);
            places[what][tid % kQnTokens] = what < 2 ? b * s.batch + at * s.token : b * s.dy_batch + at * s.dy_token;
        }
        if (p.positions)
            for (int i = tid; i < n_tokens * p.pairs; i += kBlock) {
                uint32_t t, pair;
                int b, at;
                divmod((uint32_t)i, p.by_pairs, t, pair);
                place((int)t, b, at);
                angles[i] = qn_angle<T>(p, b, at, (int)pair);
            }
        __syncthreads();
#pragma unroll
        for (int side = 0; side < 2; ++side) {
            if (gridDim.y == 2 && side != (int)blockIdx.y) continue;
            const QnSide &s = p.side[side];
            const int rows = n_tokens * s.heads;
            const T *x = reinterpret_cast<const T *>(s.x), *dy = reinterpret_cast<const T *>(s.dy);
            T *y = reinterpret_cast<T *>(s.y) + token0 * s.heads * p.dim;
            // kAhead rows of a lane on their way at once (a row's lanes are together here); past the last row that one again
            for (int row0 = slot; row0 < rows; row0 += kAhead * kSlots) {
                float v[kAhead][8], d[kBack ? kAhead : 1][8];
                uint32_t token[kAhead];
#pragma unroll
                for (int a = 0; a < kAhead; ++a) {
                    uint32_t h;
                    divmod((uint32_t)min(row0 + a * kSlots, rows - 1), p.by_heads[side], token[a], h);
                    const T *from = x + places[side][token[a]] + (int64_t)h * s.head;
                    qn_load4(from + first, v[a]);
                    qn_load4(from + second, v[a] + 4);
                    if constexpr (kBack) {
                        const T *back = dy + places[2 + side][token[a]] + (int64_t)h * s.dy_head;
                        qn_load4(back + first, d[a]);
                        qn_load4(back + second, d[a] + 4);
                    }
                }
#pragma unroll
                for (int a = 0; a < kAhead; ++a) {
                    const bool live = in && row0 + a * kSlots < rows;
                    float q = 0.0f;
#pragma unroll
                    for (int i = 0; i < 8; ++i) q = fmaf(v[a][i], v[a][i], q);
                    const float r = rsqrtf(qn_sum<kLanes>(in ? q : 0.0f) * inv_d + p.eps);
                    const float2 *cs = angles + token[a] * p.pairs + 4 * unit;
                    if constexpr (!kBack) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) v[a][i] = v[a][i] * r * w[side][i];
                        if (turned) qn_turn8(v[a], cs, p.interleaved, false);
                    } else {
                        if (turned) qn_turn8(d[a], cs, p.interleaved, true);
                        float m = 0.0f;
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            v[a][i] *= r;
                            const float g = d[a][i] * v[a][i];
                            dw[side][i] += live ? g : 0.0f;
                            d[a][i] *= w[side][i];
                            m = fmaf(d[a][i], v[a][i], m);
                        }
                        m = qn_sum<kLanes>(in ? m : 0.0f) * inv_d;
#pragma unroll
                        for (int i = 0; i < 8; ++i) v[a][i] = (d[a][i] - v[a][i] * m) * r;
                    }
                    if (live) {
                        T *to = y + (int64_t)(row0 + a * kSlots) * p.dim;
                        qn_store4(to + first, v[a]);
                        qn_store4(to + second, v[a] + 4);
                    }
                }
            }
        }
    }
    if constexpr (kBack) {
        if (!p.partial) return;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 8; ++i) sums[i * kBlock + tid] = dw[k][i];
            __syncthreads();
            if (slot == 0 && in)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    float total = 0.0f;
                    for (int j = 0; j < kSlots; ++j) total += sums[i * kBlock + j * kLanes + unit];
                    p.partial[((int64_t)blockIdx.x * 2 + k) * p.dim + (i < 4 ? first + i : second + i - 4)] = total;
                }
        }
    }
}

// Any dimension, alignment and number of pairs: a wavefront to a row, a pair or two single values to a lane at a time, the weights again for each row.
// 4 x 4096 tokens of 32 + 8 heads, bf16: of 128, one value off the grid of 8 bytes, 344 us (72 on it), with the gradients 875 (191); of 100 291 and 812.
template <typename T, bool kBack>
__global__ __launch_bounds__(kBlock) void qk_norm_rotate_any_kernel(const QnArgs p) {
    constexpr int kSlots = kBlock / kWave, kMost = kQnMaxDim / 2 / kWave;
    __shared__ float2 angles[kQnPairs];
    __shared__ float sums[kBack ? kBlock : 1];
    const int tid = threadIdx.x, slot = tid / kWave, lane = tid % kWave;
    const float inv_d = 1.0f / (float)p.dim;
    const int heads = p.side[0].heads + p.side[1].heads, units = (p.dim + 1) / 2;
    const int64_t all = (int64_t)p.batch * p.tokens;
    float dw[2][kMost][2];
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int i = 0; i < kMost; ++i) dw[k][i][0] = dw[k][i][1] = 0.0f;
    auto place = [&](int u, int which) {                             // where a unit's first and second value stand
        if (p.positions && u < p.pairs) return p.interleaved ? 2 * u + which : u + which * p.pairs;
        return 2 * u + which;                                        // (behind the 2 * pairs that turn, for u >= pairs)
    };
    for (int64_t round = blockIdx.x; round < p.rounds; round += gridDim.x) {
        const int64_t token0 = round * p.round;
        const int n_tokens = (int)(all - token0 < p.round ? all - token0 : p.round), rows = n_tokens * heads;
        if (p.positions) {
            if (round != blockIdx.x) __syncthreads();
            for (int i = tid; i < n_tokens * p.pairs; i += kBlock) {
                const int64_t token = token0 + i / p.pairs, b = token / p.tokens;
                angles[i] = qn_angle<T>(p, (int)b, (int)(token - b * p.tokens), i % p.pairs);
            }
            __syncthreads();
        }
        for (int row = slot; row < rows; row += kSlots) {
            const int t = row / heads, h = row - t * heads;
            const bool key = h >= p.side[0].heads;
            const QnSide &s = p.side[key];
            const int head = key ? h - p.side[0].heads : h;
            const int64_t token = token0 + t, b = token / p.tokens, tt = token - b * p.tokens;
            const T *x = reinterpret_cast<const T *>(s.x) + b * s.batch + tt * s.token + head * s.head;
            const T *dy = reinterpret_cast<const T *>(s.dy) + b * s.dy_batch + tt * s.dy_token + head * s.dy_head;
            float v[kMost][2], d[kMost][2], w[kMost][2], q = 0.0f;
#pragma unroll
            for (int i = 0; i < kMost; ++i)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int u = lane + i * kWave, at = place(u, e);
                    const bool in = u < units && at < p.dim;
                    v[i][e] = in ? to_f32(x[at]) : 0.0f;
                    w[i][e] = in ? qn_weight(s.w, at, p.w_dtype) : 0.0f;
                    d[i][e] = kBack && in ? to_f32(dy[at]) : 0.0f;
                    q = fmaf(v[i][e], v[i][e], q);
                }
            const float r = rsqrtf(qn_sum<kWave>(q) * inv_d + p.eps);
            float m = 0.0f;
#pragma unroll
            for (int i = 0; i < kMost; ++i) {
                const int u = lane + i * kWave;
                const bool turned = p.positions && u < p.pairs;
                if constexpr (kBack) {
                    if (turned) qn_turn(d[i][0], d[i][1], angles[t * p.pairs + u], true);
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        v[i][e] *= r;
                        const float g = d[i][e] * v[i][e];
                        dw[0][i][e] += key ? 0.0f : g;
                        dw[1][i][e] += key ? g : 0.0f;
                        d[i][e] *= w[i][e];
                        m = fmaf(d[i][e], v[i][e], m);
                    }
                } else {
                    v[i][0] *= r * w[i][0];
                    v[i][1] *= r * w[i][1];
                    if (turned) qn_turn(v[i][0], v[i][1], angles[t * p.pairs + u], false);
                }
            }
            if constexpr (kBack) {
                m = qn_sum<kWave>(m) * inv_d;
#pragma unroll
                for (int i = 0; i < kMost; ++i)
#pragma unroll
                    for (int e = 0; e < 2; ++e) v[i][e] = (d[i][e] - v[i][e] * m) * r;
            }
            T *y = reinterpret_cast<T *>(s.y) + (token * s.heads + head) * p.dim;
#pragma unroll
            for (int i = 0; i < kMost; ++i)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int u = lane + i * kWave, at = place(u, e);
                    if (u < units && at < p.dim) y[at] = from_f32<T>(v[i][e]);
                }
        }
    }
    if constexpr (kBack) {
        if (!p.partial) return;
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int i = 0; i < kMost; ++i)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    __syncthreads();
                    sums[tid] = dw[k][i][e];
                    __syncthreads();
                    const int u = lane + i * kWave, at = place(u, e);
                    if (slot == 0 && u < units && at < p.dim)
                        p.partial[((int64_t)blockIdx.x * 2 + k) * p.dim + at] = (sums[lane] + sums[kWave + lane]) + (sums[2 * kWave + lane] + sums[3 * kWave + lane]);
                }
    }
}

// The workgroups' sums of the weights' gradients: 16 columns to a workgroup, the shares dealt out to its 64 slots
__global__ __launch_bounds__(1024) void qn_weights_kernel(const float *partial, void *dqw, void *dkw, int shares, int dim, int dtype) {
    __shared__ float sums[64][17];
    const int slot = threadIdx.x / 16, at = threadIdx.x % 16, col = blockIdx.x * 16 + at, safe = min(col, 2 * dim - 1);
    float total = 0.0f;
#pragma unroll 4
    for (int s = slot; s < shares; s += 64) total += partial[(int64_t)s * 2 * dim + safe];
    sums[slot][at] = total;
    for (int d = 32; d >= 1; d /= 2) {
        __syncthreads();
        if (slot < d) sums[slot][at] += sums[slot + d][at];
    }
    if (slot != 0 || col >= 2 * dim) return;
    total = sums[0][at];
    void *out = col < dim ? dqw : dkw;
    const int place = col < dim ? col : col - dim;
    if (!out) return;
    if (dtype == SS2D_F32) reinterpret_cast<float *>(out)[place] = total;
    else if (dtype == SS2D_BF16) reinterpret_cast<bf16_t *>(out)[place] = from_f32<bf16_t>(total);
    else reinterpret_cast<f16_t *>(out)[place] = from_f32<f16_t>(total);
}

static int qn_arguments(const ss2d_qk_norm_rotate_params *p, QnArgs &a, bool &vec, bool back, const ss2d_qk_norm_rotate_bwd_params *g) {
    if (!p) return SS2D_EINVAL;
    if (p->batch < 0 || p->seqlen < 0 || p->q_heads < 0 || p->k_heads < 0 || p->dim < 1 || p->dtype < SS2D_F32 || p->dtype > SS2D_F16) return SS2D_EINVAL;
    if ((p->q_weight || p->k_weight) && p->weight_dtype != SS2D_F32 && p->weight_dtype != p->dtype) return SS2D_EINVAL;
    if (p->dim > kQnMaxDim || p->seqlen > 0x7fffffff - kQnTokens) return SS2D_ENOTSUP;       // (a round's tokens are counted on from its first one's place)
    a = {};
    if (p->positions) {
        if (!p->frequencies || p->axes < 1 || p->per_axis < 1 || p->per_axis > p->dim || p->axes > p->dim || 2 * p->axes * p->per_axis > p->dim) return SS2D_EINVAL;
        a.axes = p->axes; a.per_axis = p->per_axis; a.pairs = p->axes * p->per_axis;
        a.positions = p->positions; a.frequencies = p->frequencies; a.pos64 = p->positions_int64; a.freq64 = p->frequencies_float64;
        a.pos_batch = p->position_batch_stride; a.pos_token = p->position_token_stride; a.pos_axis = p->position_axis_stride;
    }
    a.batch = p->batch; a.tokens = p->seqlen; a.dim = p->dim; a.w_dtype = p->weight_dtype; a.interleaved = p->interleaved != 0; a.eps = p->eps;
    a.side[0] = {p->q, nullptr, p->q_out, p->q_weight, p->q_batch_stride, p->q_token_stride, p->q_head_stride, 0, 0, 0, p->q_heads};
    a.side[1] = {p->k, nullptr, p->k_out, p->k_weight, p->k_batch_stride, p->k_token_stride, p->k_head_stride, 0, 0, 0, p->k_heads};
    if (back) {
        a.side[0].dy = g->dq_out; a.side[0].y = g->dq;
        a.side[0].dy_batch = g->dq_batch_stride; a.side[0].dy_token = g->dq_token_stride; a.side[0].dy_head = g->dq_head_stride;
        a.side[1].dy = g->dk_out; a.side[1].y = g->dk;
        a.side[1].dy_batch = g->dk_batch_stride; a.side[1].dy_token = g->dk_token_stride; a.side[1].dy_head = g->dk_head_stride;
    }
    vec = p->dim % 8 == 0 && 2 * a.pairs % 8 == 0;
    const int64_t size = p->dtype == SS2D_F32 ? 4 : 2;
    for (const QnSide &s : a.side) {
        if (s.w && (uintptr_t)s.w % (p->weight_dtype == SS2D_F32 ? 16 : 8) != 0) vec = false;
        if (s.heads == 0) continue;
        uintptr_t bits = (uintptr_t)s.x | (uintptr_t)s.y | (uintptr_t)(s.batch * size) | (uintptr_t)(s.token * size) | (uintptr_t)(s.head * size);
        if (back) bits |= (uintptr_t)s.dy | (uintptr_t)(s.dy_batch * size) | (uintptr_t)(s.dy_token * size) | (uintptr_t)(s.dy_head * size);
        vec = vec && bits % (4 * size) == 0;
    }
    const int64_t all = (int64_t)a.batch * a.tokens, heads = (int64_t)p->q_heads + p->k_heads;
    if (heads > 0x7fffffff / kQnTokens / kQnMaxDim) return SS2D_EINVAL;
    // A round's rows come to a group of lanes `ahead` at a time: as many tokens as make these full on both sides, while a thousand workgroups remain
    int lanes = 4;
    while (8 * lanes < p->dim) lanes *= 2;
    const int64_t step = (int64_t)(kBlock / (vec ? lanes : kWave)) * (!vec ? 1 : back ? 2 : 4);
    int64_t most = kQnTokens, round = 1;
    if (a.pairs > 0 && most > kQnPairs / a.pairs) most = kQnPairs / a.pairs;
    double best = 0.0;
    for (int64_t n = 1; n <= most && (n == 1 || all / n >= 1024); ++n) {
        double rows = 0.0, taken = 0.0;
        for (const QnSide &s : a.side) {
            rows += (double)(n * s.heads);
            taken += (double)((n * s.heads + step - 1) / step * step);
        }
        const double full = rows / (taken + step);                   // (and a step's worth for the angles)
        if (full > best) { best = full; round = n; }
    }
    a.round = (int)round;
    for (int i = 0; i < 2; ++i) a.by_heads[i] = make_fastdiv((uint32_t)(a.side[i].heads > 0 ? a.side[i].heads : 1));
    a.by_pairs = make_fastdiv((uint32_t)(a.pairs > 0 ? a.pairs : 1));
    a.by_tokens = make_fastdiv((uint32_t)(a.tokens > 0 ? a.tokens : 1));
    a.rounds = all > 0 && heads > 0 ? (all + round - 1) / round : 0;
    return SS2D_OK;
}

constexpr int64_t kQnShares = 1024;                                  // workgroups of the backward: four to a CU
constexpr int64_t kQnGrid = 1 << 22;                                 // of the forward (a launch's threads fit 32 bits)

template <typename T, bool kBack> static int qn_launch(const QnArgs &a, bool vec, uint32_t shares, hipStream_t st) {
    // few rounds (a workgroup to a CU at most): queries and keys to workgroups of their own, one after the other they take longer
    const dim3 grid(shares, !kBack && vec && shares <= 256 ? 2 : 1);
    if (!vec) qk_norm_rotate_any_kernel<T, kBack><<<grid, kBlock, 0, st>>>(a);
    else if (a.dim <= 32) qk_norm_rotate_kernel<T, 4, kBack><<<grid, kBlock, 0, st>>>(a);
    else if (a.dim <= 64) qk_norm_rotate_kernel<T, 8, kBack><<<grid, kBlock, 0, st>>>(a);
    else if (a.dim <= 128) qk_norm_rotate_kernel<T, 16, kBack><<<grid, kBlock, 0, st>>>(a);
    else if (a.dim <= 256) qk_norm_rotate_kernel<T, 32, kBack><<<grid, kBlock, 0, st>>>(a);
    else qk_norm_rotate_kernel<T, 64, kBack><<<grid, kBlock, 0, st>>>(a);
    return launch_status();
}

}  // namespace ss2d

using namespace ss2d;

extern "C" int ss2d_qk_norm_rotate(const ss2d_qk_norm_rotate_params *p, void *stream) {
    QnArgs a;
    bool vec;
    const int rc = qn_arguments(p, a, vec, false, nullptr);
    if (rc != SS2D_OK || a.rounds == 0) return rc;
    if ((p->q_heads && (!p->q || !p->q_out)) || (p->k_heads && (!p->k || !p->k_out))) return SS2D_EINVAL;
    const uint32_t grid = (uint32_t)(a.rounds < kQnGrid ? a.rounds : kQnGrid);
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    switch (p->dtype) {
    case SS2D_F32: return qn_launch<float, false>(a, vec, grid, st);
    case SS2D_BF16: return qn_launch<bf16_t, false>(a, vec, grid, st);
    default: return qn_launch<f16_t, false>(a, vec, grid, st);
    }
}

extern "C" int64_t ss2d_qk_norm_rotate_bwd_workspace_bytes(int dim) { return dim > 0 && dim <= kQnMaxDim ? kQnShares * 2 * dim * (int64_t)sizeof(float) : SS2D_EINVAL; }

extern "C" int ss2d_qk_norm_rotate_bwd(const ss2d_qk_norm_rotate_bwd_params *g, void *workspace, int64_t workspace_bytes, void *stream) {
    if (!g) return SS2D_EINVAL;
    const ss2d_qk_norm_rotate_params *p = &g->fwd;
    QnArgs a;
    bool vec;
    const int rc = qn_arguments(p, a, vec, true, g);
    if (rc != SS2D_OK) return rc;
    if ((g->dq_weight && !p->q_weight) || (g->dk_weight && !p->k_weight)) return SS2D_EINVAL;
    const bool weights = g->dq_weight || g->dk_weight;
    if (a.rounds && ((p->q_heads && (!p->q || !g->dq_out || !g->dq)) || (p->k_heads && (!p->k || !g->dk_out || !g->dk)))) return SS2D_EINVAL;
    if (weights) {
        if (!workspace || (uintptr_t)workspace % 16 != 0) return SS2D_EINVAL;
        if (workspace_bytes < ss2d_qk_norm_rotate_bwd_workspace_bytes(p->dim)) return SS2D_ENOMEM;
        a.partial = reinterpret_cast<float *>(workspace);
    }
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    const uint32_t grid = (uint32_t)(a.rounds < kQnShares ? a.rounds : kQnShares);
    if (grid) {
        int status;
        switch (p->dtype) {
        case SS2D_F32: status = qn_launch<float, true>(a, vec, grid, st); break;
        case SS2D_BF16: status = qn_launch<bf16_t, true>(a, vec, grid, st); break;
        default: status = qn_launch<f16_t, true>(a, vec, grid, st);
        }
        if (status != SS2D_OK) return status;
    }
    if (weights) qn_weights_kernel<<<(2 * p->dim + 15) / 16, 1024, 0, st>>>(a.partial, g->dq_weight, g->dk_weight, (int)grid, p->dim, p->weight_dtype);
    return launch_status();
}
