// One token of linear attention with a decay for each head, the state updated in place:
//     S = exp(g) S + k v^T,   o = scale q^T S.
// The state is read and written once and everything else is small, so memory bounds it: 8 bytes per value of the state.  A
// workgroup owns some columns (values) of one head's state for all keys; a row of them is kVec floats to a lane, all rows of a
// round on their way at once, and the lanes' sums meet in LDS.  256 sequences, 32 heads of 128 x 128: 182 us for 1.08 GB, 5.9 TB/s (a copy's rate is 5.3).  One
// sequence, 8 heads of 64 x 64: 5.2 us, a launch and two trips to memory, in workgroups of 16 columns.
#include "linear_attention.h"

namespace ss2d {

struct LaStepArgs {
    LaSide q, k, v;                  // (token stride unused)
    const void *decay;
    int64_t decay_batch, decay_head;
    int32_t decay_dtype, heads;
    float *state;
    int64_t state_batch;
    void *out;                       // (batch, heads, Dv), dense
    float scale;
};

constexpr int kStepRows = 8;         // of the state, loads in flight to a lane

// kVec values to a lane, kCols columns to a workgroup
template <typename T, int kVec, int kCols>
__global__ __launch_bounds__(kBlock) void la_step_kernel(const LaStepArgs p, int tiles) {
    constexpr int kLanes = kCols / kVec, kSlots = kBlock / kLanes;   // lanes of a row, rows of a round
    __shared__ float qs[kLaMaxDim], ks[kLaMaxDim], sums[kSlots][kCols];
    typedef float vec_t __attribute__((ext_vector_type(kVec)));
    const int tid = threadIdx.x, slot = tid / kLanes, at = tid % kLanes * kVec;
    const int tile = blockIdx.x % (uint32_t)tiles, h = blockIdx.x / (uint32_t)tiles % (uint32_t)p.heads;
    const int64_t b = blockIdx.x / (uint32_t)tiles / (uint32_t)p.heads;
    const int dk = p.k.dim, dv = p.v.dim, c = tile * kCols + at;
    const bool in = c < dv;                                          // (kVec divides dv)
    if (tid < dk) {
        qs[tid] = to_f32(reinterpret_cast<const T *>(p.q.p)[b * p.q.batch + (int64_t)(h / p.q.div) * p.q.head + tid]);
        ks[tid] = to_f32(reinterpret_cast<const T *>(p.k.p)[b * p.k.batch + (int64_t)(h / p.k.div) * p.k.head + tid]);
    }
    const float decay = p.decay ? __expf(load_decay(p.decay, b * p.decay_batch + h * p.decay_head, p.decay_dtype)) : 1.0f;
    float *state = p.state + b * p.state_batch + (int64_t)h * dk * dv + c;
    vec_t v, sum;
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
        v[i] = in ? to_f32(reinterpret_cast<const T *>(p.v.p)[b * p.v.batch + (int64_t)(h / p.v.div) * p.v.head + c + i]) : 0.0f;
        sum[i] = 0.0f;
    }
    auto fetch = [&](int r0, vec_t (&s)[kStepRows]) {                // (rows past the last repeat it, columns past theirs the first; nobody stores them)
#pragma unroll
        for (int i = 0; i < kStepRows; ++i) s[i] = load_streaming(reinterpret_cast<const vec_t *>(state + (in ? 0 : -c) + (int64_t)min(r0 + slot + i * kSlots, dk - 1) * dv));
    };
    vec_t s[kStepRows];
    fetch(0, s);
    __syncthreads();
    for (int r0 = 0; r0 < dk; r0 += kStepRows * kSlots) {
        if (r0) fetch(r0, s);
#pragma unroll
        for (int i = 0; i < kStepRows; ++i) {
            const int r = r0 + slot + i * kSlots;
            const float key = r < dk ? ks[r] : 0.0f;
            s[i] = s[i] * decay + v * key;
            if (in && r < dk) {
                store_streaming(reinterpret_cast<vec_t *>(state + (int64_t)r * dv), s[i]);
                sum += s[i] * qs[r];
            }
        }
    }
#pragma unroll
    for (int i = 0; i < kVec; ++i) sums[slot][at + i] = sum[i];
    __syncthreads();
    if (tid < kCols && tile * kCols + tid < dv) {
        float total = 0.0f;
#pragma unroll
        for (int i = 0; i < kSlots; ++i) total += sums[i][tid];
        reinterpret_cast<T *>(p.out)[(b * p.heads + h) * dv + tile * kCols + tid] = from_f32<T>(total * p.scale);
    }
}

template <typename T> static int la_step(const LaStepArgs &a, int batch, hipStream_t stream) {
    const int dv = a.v.dim;
    const int64_t heads = (int64_t)batch * a.heads;
    const bool vec = dv % 4 == 0 && (uintptr_t)a.state % 16 == 0 && a.state_batch % 4 == 0;
    auto go = [&](auto kernel, int cols) {
        const int64_t tiles = (dv + cols - 1) / cols, total = heads * tiles;
        if (total > kLaLaunch / kBlock) return (int)SS2D_ENOTSUP;
        kernel<<<(uint32_t)total, kBlock, 0, stream>>>(a, (int)tiles);
        return launch_status();
    };
    if (!vec) return go(la_step_kernel<T, 1, 16>, 16);
    // few heads: more workgroups of fewer columns
    return heads * ((dv + 63) / 64) >= 512 ? go(la_step_kernel<T, 4, 64>, 64) : go(la_step_kernel<T, 4, 16>, 16);
}

LaSide la_side(const void *ptr, int64_t batch, int64_t token, int64_t head, int heads, int own_heads, int dim, int size);

}  // namespace ss2d

using namespace ss2d;

extern "C" int ss2d_linear_attention_step(const ss2d_linear_attention_step_params *p, void *stream) {
    if (!p || p->batch < 0 || p->heads < 0 || p->key_dim < 1 || p->value_dim < 1 || p->q_heads < 1 || p->k_heads < 1 || p->v_heads < 1) return SS2D_EINVAL;
    if (p->dtype < SS2D_F32 || p->dtype > SS2D_F16 || (p->decay && p->decay_dtype != SS2D_F32 && p->decay_dtype != p->dtype)) return SS2D_EINVAL;
    if (p->heads % p->q_heads || p->heads % p->k_heads || p->heads % p->v_heads) return SS2D_EINVAL;
    if (p->key_dim > kLaMaxDim || p->value_dim > kLaMaxDim) return SS2D_ENOTSUP;
    if (p->batch == 0 || p->heads == 0) return SS2D_OK;
    if (!p->q || !p->k || !p->v || !p->state || !p->out) return SS2D_EINVAL;
    if (p->batch > 1 && p->state_batch_stride < (int64_t)p->heads * p->key_dim * p->value_dim) return SS2D_EINVAL;
    LaStepArgs a = {};
    a.q = la_side(p->q, p->q_batch_stride, 0, p->q_head_stride, p->heads, p->q_heads, p->key_dim, 1);
    a.k = la_side(p->k, p->k_batch_stride, 0, p->k_head_stride, p->heads, p->k_heads, p->key_dim, 1);
    a.v = la_side(p->v, p->v_batch_stride, 0, p->v_head_stride, p->heads, p->v_heads, p->value_dim, 1);
    a.decay = p->decay; a.decay_dtype = p->decay_dtype; a.decay_batch = p->decay_batch_stride; a.decay_head = p->decay_head_stride;
    a.heads = p->heads; a.state = p->state; a.state_batch = p->state_batch_stride; a.out = p->out; a.scale = p->scale;
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    switch (p->dtype) {
    case SS2D_F32: return la_step<float>(a, p->batch, st);
    case SS2D_F16: return la_step<f16_t>(a, p->batch, st);
    default: return la_step<bf16_t>(a, p->batch, st);
    }
}
