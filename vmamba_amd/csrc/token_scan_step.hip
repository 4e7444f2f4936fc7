// One token of the selective scan of token sequences, the states updated in place (token_scan.h has the formulas):
//     h = exp(step A) h + step u B,   y = (C . h + D u) silu(z).
// The states are read and written once and everything else is small, so memory bounds it: 8 bytes per value of a state.  Four states to a lane, a
// channel's lanes side by side; a workgroup's channels are taken for kRows sequences at once, so that A and the channels' constants are read once for
// them and several states are on their way.  256 sequences of 4096 channels and 16 states: 23 us, 5.9 TB/s.
#include "token_scan.h"

namespace ss2d {

struct TsStepArgs {
    const void *u, *delta, *B, *C, *z;
    const float *A, *D, *bias;
    float *state;
    void *out;
    int64_t u_b, dl_b, z_b, B_b, B_g, C_b, C_g, state_b;
    int32_t batch, dim, N, per_group, softplus;
};

template <typename T, int kLanes, int kRows>
__global__ __launch_bounds__(kBlock) void ts_step_kernel(const TsStepArgs p, uint32_t blocks) {
    constexpr int kChans = kBlock / kLanes;
    typedef float here __attribute__((ext_vector_type(4), aligned(4)));
    const int lane = threadIdx.x % kLanes, d0 = (int)(blockIdx.x % blocks) * kChans + (int)threadIdx.x / kLanes, d = min(d0, p.dim - 1), n = 4 * lane;
    const int64_t b0 = (int64_t)(blockIdx.x / blocks) * kRows;
    const bool whole = n + 4 <= p.N, any = n < p.N;
    const int g = d / p.per_group;
    floatx4_t h[kRows];
    float uv[kRows], dv[kRows], zv[kRows], Bv[kRows][4], Cv[kRows][4];
    auto four = [&](const float *from) {
        if (whole) return (floatx4_t) * reinterpret_cast<const here *>(from + n);
        floatx4_t v = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < 3; ++i)
            if (n + i < p.N) v[i] = from[n + i];
        return v;
    };
#pragma unroll
    for (int r = 0; r < kRows; ++r) {                                // (sequences past the last repeat it; nobody stores them)
        const int64_t b = min(b0 + r, (int64_t)p.batch - 1);
        h[r] = four(p.state + b * p.state_b + (int64_t)d * p.N);
        uv[r] = to_f32(((const T *)p.u)[b * p.u_b + d]);
        dv[r] = to_f32(((const T *)p.delta)[b * p.dl_b + d]);
        zv[r] = p.z ? to_f32(((const T *)p.z)[b * p.z_b + d]) : 0.0f;
        const int have = min(max(p.N - n, 0), 4);
        ts_widen<T>(ts_load4<T>((const T *)p.B + b * p.B_b + g * p.B_g + (any ? n : 0), have, p.N == 4 * kLanes), Bv[r]);
        ts_widen<T>(ts_load4<T>((const T *)p.C + b * p.C_b + g * p.C_g + (any ? n : 0), have, p.N == 4 * kLanes), Cv[r]);
    }
    const floatx4_t A2 = four(p.A + (int64_t)d * p.N) * kLog2e;
    const float bias = p.bias ? p.bias[d] : 0.0f, skip = p.D ? p.D[d] : 0.0f;
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
        const float step = p.softplus ? softplus_log2(fmaf(dv[r], kLog2e, bias * kLog2e)) : dv[r] + bias, fed = step * uv[r];
        float y = 0.0f;
#pragma unroll
        for (int v = 0; v < 4; ++v) {
            h[r][v] = fmaf(fed, Bv[r][v], __builtin_amdgcn_exp2f(step * A2[v]) * h[r][v]);
            y = fmaf(Cv[r][v], h[r][v], y);
        }
        if (!whole) {                                                // (states that are not there: whatever the step is, they add nothing)
            y = 0.0f;
#pragma unroll
            for (int v = 0; v < 3; ++v)
                if (n + v < p.N) y = fmaf(Cv[r][v], h[r][v], y);
        }
#pragma unroll
        for (int over = 1; over < kLanes; over *= 2) y += __shfl_xor(y, over, kWave);
        if (b0 + r >= p.batch || d0 >= p.dim) continue;
        float *to = p.state + (b0 + r) * p.state_b + (int64_t)d * p.N;
        if (whole) *reinterpret_cast<here *>(to + n) = h[r];
        else
#pragma unroll
            for (int v = 0; v < 3; ++v)
                if (n + v < p.N) to[n + v] = h[r][v];
        if (lane == 0) {
            y = p.D ? fmaf(skip, uv[r], y) : y;
            ((T *)p.out)[(b0 + r) * p.dim + d] = from_f32<T>(p.z ? y * (zv[r] * ts_sigmoid(zv[r])) : y);
        }
    }
}

template <typename T, int kLanes> static int ts_step(const TsStepArgs &a, hipStream_t st) {
    constexpr int kChans = kBlock / kLanes;
    const int64_t blocks = (a.dim + kChans - 1) / kChans;
    auto go = [&](auto kernel, int rows) {
        const int64_t n = blocks * (((int64_t)a.batch + rows - 1) / rows);
        if (n > kTsLaunch / kBlock) return (int)SS2D_ENOTSUP;
        kernel<<<(uint32_t)n, kBlock, 0, st>>>(a, (uint32_t)blocks);
        return launch_status();
    };
    // (2048 channels of 16 states, four sequences to a workgroup and one: 64 sequences 7.1 to 7.3 us either way, 96 8.0; 128, from where on, 8.9 and 9.3; 256 14.5 and 16.6)
    return blocks * a.batch >= 4096 ? go(ts_step_kernel<T, kLanes, 4>, 4) : go(ts_step_kernel<T, kLanes, 1>, 1);
}

}  // namespace ss2d

using namespace ss2d;

extern "C" int ss2d_token_scan_step(const ss2d_token_scan_step_params *p, void *stream) {
    if (!p || p->batch < 0 || p->dim < 0 || p->dstate < 1 || p->n_groups < 1 || p->dim % p->n_groups) return SS2D_EINVAL;
    if (p->dtype < SS2D_F32 || p->dtype > SS2D_F16) return SS2D_EINVAL;
    if (p->dstate > kTsMaxState || p->dim > INT32_MAX - kBlock) return SS2D_ENOTSUP;    // (a workgroup's last channels are counted in 32 bits)
    if (p->batch == 0 || p->dim == 0) return SS2D_OK;
    if (!p->u || !p->delta || !p->A || !p->B || !p->C || !p->state || !p->out) return SS2D_EINVAL;
    if (p->batch > 1 && p->state_batch_stride < (int64_t)p->dim * p->dstate) return SS2D_EINVAL;
    const TsStepArgs a = {p->u, p->delta, p->B, p->C, p->z, p->A, p->D, p->delta_bias, p->state, p->out, p->u_batch_stride, p->delta_batch_stride, p->z_batch_stride,
                          p->B_batch_stride, p->B_group_stride, p->C_batch_stride, p->C_group_stride, p->state_batch_stride, p->batch, p->dim, p->dstate,
                          p->dim / p->n_groups, p->delta_softplus != 0};
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    auto with = [&](auto t) {
        using T = decltype(t);
        if (a.N <= 4) return ts_step<T, 1>(a, st);
        if (a.N <= 8) return ts_step<T, 2>(a, st);
        if (a.N <= 16) return ts_step<T, 4>(a, st);
        return a.N <= 32 ? ts_step<T, 8>(a, st) : ts_step<T, 16>(a, st);
    };
    return p->dtype == SS2D_F32 ? with(float{}) : p->dtype == SS2D_F16 ? with(f16_t{}) : with(bf16_t{});
}
