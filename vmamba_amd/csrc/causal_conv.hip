// The short causal convolution of token sequences, each channel for itself, with its gradients and its form for single tokens:
//     y_t = act(bias + sum_j w_j x_(t - W + 1 + j)),   act = SiLU or none; what is before a sequence's first token is its state, the last W - 1 inputs.
// With g_t = dout_t act'(..):   dx_t = sum_j w_j g_(t + W - 1 - j),   dw_j = sum over t of g_t x_(t - W + 1 + j),   dbias = sum g.
//
// Memory bounds it: 8 x 4096 tokens of 2048 channels in bf16 61 us (4.4 TB/s; a strip of 32 tokens 65, of 128 67), their gradients 90 (4.5 TB/s) and 6 for the sums over strips;
// from the caches, which hold half of it, 44 and 80.
// A thread takes the channels of one 16-byte piece (of few tokens: two channels) and walks a strip of tokens with the window in registers; rows are
// loaded a chunk at a time, all on their way at once.  Threads side by side have neighbouring pieces, strips below each other.  The last
// piece of a row ends with it, so that it may repeat channels of the one before: both write the same values.
#include "row_piece.h"
#include "token_scan.h"

namespace ss2d {

struct CvArgs {
    const void *x, *weight, *bias, *initial;
    const int32_t *cu;
    void *out, *final;
    int64_t x_b, x_t;
    int32_t batch, tokens, dim, n_seqs, silu, weight_f32;
    int32_t near;                    // every tensor's bytes are counted by 32 bits: a row is a uniform place and a lane's offset
    int32_t pieces, cols, piece_blocks, strip, strips;               // cols: pieces side by side in a workgroup; strips of a row
    // gradients
    const void *dout, *dfinal;
    void *dx, *dinitial;
    int64_t do_b, do_t;
    float *sums;                                                     // [strips of a workgroup][w_0 .. w_(W-1), bias][channel]
};

// The weights of kV channels: w[j][i] of channel i, and the bias
template <typename T, int kW, int kV> __device__ __forceinline__ void cv_weights(const CvArgs &p, int d, float (&w)[kW][kV], float (&bias)[kV]) {
    auto read = [&](auto t) {
        using U = decltype(t);
        const U *from = (const U *)p.weight + (int64_t)d * kW, *b = (const U *)p.bias + d;
#pragma unroll
        for (int k = 0; k < kW; ++k) {                               // (channel, tap) is dense
            const RowPiece<U, kV> r = load_row_piece<U, kV>(from + k * kV);
#pragma unroll
            for (int i = 0; i < kV; ++i) w[(k * kV + i) % kW][(k * kV + i) / kW] = r.get(i);
        }
        if (p.bias) {
            const RowPiece<U, kV> r = load_row_piece<U, kV>(b);
#pragma unroll
            for (int i = 0; i < kV; ++i) bias[i] = r.get(i);
        } else {
#pragma unroll
            for (int i = 0; i < kV; ++i) bias[i] = 0.0f;
        }
    };
    if (p.weight_f32) read(float{});
    else read(T{});
}

struct CvPlace { int b, t0, t1, d, strip; bool there; };

// What a thread of a grid of strips and pieces does
template <int kV> __device__ __forceinline__ CvPlace cv_place(const CvArgs &p, uint32_t &group) {
    const uint32_t id = xcd_contiguous_id(blockIdx.x, gridDim.x);
    group = id / (uint32_t)p.piece_blocks;
    const int piece = (int)(id % (uint32_t)p.piece_blocks) * p.cols + (int)threadIdx.x % p.cols;
    const int64_t s = (int64_t)group * (kBlock / p.cols) + (int)threadIdx.x / p.cols;
    CvPlace c;
    c.there = piece < p.pieces && s < (int64_t)p.batch * p.strips;
    c.b = c.there ? (int)(s / p.strips) : 0;
    c.strip = c.there ? (int)(s % p.strips) : 0;
    c.t0 = c.strip * p.strip;
    c.t1 = min(c.t0 + p.strip, p.tokens);
    c.d = min(piece * kV, p.dim - kV);
    return c;
}

// The value behind token `t` of the line (state, then inputs) of a sequence: t >= lo - W + 1
template <typename T, int kW, int kV> __device__ __forceinline__ RowPiece<T, kV> cv_line(const CvArgs &p, const T *x, const TsSpan &sp, int d, int t) {
    if (t >= sp.lo) return load_row_piece<T, kV>(x + (int64_t)t * p.x_t);
    RowPiece<T, kV> r = {};
    if (p.initial) r = load_row_piece<T, kV>((const T *)p.initial + ((int64_t)sp.seq * (kW - 1) + (t - sp.lo + kW - 1)) * p.dim + d);
    return r;
}

template <typename T, int kV> __device__ __forceinline__ void cv_copy_row(const T *from, T *to) {
    float v[kV] = {};
    if (from) {
        const RowPiece<T, kV> r = load_row_piece<T, kV>(from);
#pragma unroll
        for (int i = 0; i < kV; ++i) v[i] = r.get(i);
    }
    store_row_piece<T, kV>(to, v);
}

constexpr int kCvRows = 8;           // rows of a chunk
// Values of a forward below which a thread takes two channels and four rows: its instructions are a quarter, and where every wavefront runs once, fetching them is what
// it waits for.  37 tokens of 1024 channels 5.1 -> 3.0 us, 8 x 512 of 2048 (2^23) 14.5 -> 12.7; twice as many 18.4, and 23.2 by that form.
constexpr int64_t kCvFew = 1 << 23;
constexpr int kCvFewRows = 4;

// Rows of a tensor from a lane's first one on.  at(): a row that is as far on in every lane (kNear: a uniform address, and the lane's offset, which costs no vector
// instruction); any(): one that is not.
template <typename T, bool kNear> struct CvRow {
    const T *base;
    int64_t stride;
    uint32_t off;
    __device__ __forceinline__ CvRow(const void *p, int64_t stride_, int64_t first) : base((const T *)p), stride(stride_), off(0) {
        if constexpr (kNear) off = (uint32_t)first * (uint32_t)sizeof(T);
        else base += first;
    }
    __device__ __forceinline__ const T *at(int k) const { return reinterpret_cast<const T *>(reinterpret_cast<const char *>(base + k * stride) + off); }
    __device__ __forceinline__ const T *any(int k) const {
        if constexpr (kNear) return reinterpret_cast<const T *>(reinterpret_cast<const char *>(base) + (off + (uint32_t)k * (uint32_t)(stride * (int64_t)sizeof(T))));
        return base + k * stride;
    }
};

template <typename T, int kW, int kV, bool kNear, int kRows> __global__ __launch_bounds__(kBlock) void cv_kernel(const CvArgs p) {
    uint32_t group;
    const CvPlace c = cv_place<kV>(p, group);
    if (!c.there) return;
    const T *x = (const T *)p.x + (int64_t)c.b * p.x_b + c.d;
    T *out = (T *)p.out + (int64_t)c.b * p.tokens * p.dim + c.d, *final = (T *)p.final + c.d;
    const int64_t state = (int64_t)(kW - 1) * p.dim;
    float w[kW][kV], bias[kV];
    bool read = false;
    if (p.cu && p.final)                                             // sequences without tokens, dealt out over the strips
        for (uint32_t i = c.strip; i < (uint32_t)p.n_seqs; i += p.strips)
            if (min(max(p.cu[i + 1], 0), p.tokens) <= min(max(p.cu[i], 0), p.tokens))
                for (int r = 0; r < kW - 1; ++r) cv_copy_row<T, kV>(p.initial ? (const T *)p.initial + i * state + r * (int64_t)p.dim + c.d : nullptr, final + i * state + r * (int64_t)p.dim);
    for (int a = c.t0; a < c.t1;) {
        const TsSpan sp = ts_span_at(p.cu, p.n_seqs, p.tokens, c.b, a);
        const int e = min(sp.hi, c.t1);
        if (sp.seq < 0) {                                            // tokens of no sequence
            for (int t = a; t < e; ++t) cv_copy_row<T, kV>(nullptr, out + (int64_t)t * p.dim);
            a = e;
            continue;
        }
        RowPiece<T, kV> before[kW - 1], rows[kRows];
#pragma unroll
        for (int r = 0; r < kW - 1; ++r) before[r] = cv_line<T, kW, kV>(p, x, sp, c.d, a - kW + 1 + r);
        const CvRow<T, kNear> x_row(p.x, p.x_t, c.b * p.x_b + a * p.x_t + c.d), out_row(p.out, p.dim, ((int64_t)c.b * p.tokens + a) * p.dim + c.d);
        auto request = [&](int i0) {                                 // (as many tokens on in every lane)
            const bool whole = a + i0 + kRows <= e;
#pragma unroll
            for (int k = 0; k < kRows; ++k) rows[k] = load_row_piece<T, kV>(whole ? x_row.at(i0 + k) : x_row.any(min(i0 + k, e - 1 - a)));
        };
        request(0);
        if (!read) cv_weights<T, kW, kV>(p, c.d, w, bias);           // (on their way with the first rows: 37 tokens are one latency)
        read = true;
        float window[kW - 1][kV];
#pragma unroll
        for (int r = 0; r < kW - 1; ++r)
#pragma unroll
            for (int i = 0; i < kV; ++i) window[r][i] = before[r].get(i);
        for (int i0 = 0;;) {
            const int t = a + i0;
            const bool whole = t + kRows <= e;
#pragma unroll
            for (int k = 0; k < kRows; ++k) {
                float y[kV];
#pragma unroll
                for (int i = 0; i < kV; ++i) {
                    const float now = rows[k].get(i);
                    y[i] = fmaf(w[kW - 1][i], now, bias[i]);
#pragma unroll
                    for (int j = 0; j < kW - 1; ++j) y[i] = fmaf(w[j][i], window[j][i], y[i]);
#pragma unroll
                    for (int j = 0; j < kW - 2; ++j) window[j][i] = window[j + 1][i];
                    window[kW - 2][i] = now;
                    if (p.silu) y[i] *= ts_sigmoid(y[i]);
                }
                if (whole || t + k < e) store_row_piece<T, kV>(const_cast<T *>(out_row.at(i0 + k)), y);
            }
            i0 += kRows;
            if (a + i0 >= e) break;
            request(i0);
        }
        if (e == sp.hi && p.final) {
#pragma unroll
            for (int r = 0; r < kW - 1; ++r) before[r] = cv_line<T, kW, kV>(p, x, sp, c.d, e - kW + 1 + r);
#pragma unroll
            for (int r = 0; r < kW - 1; ++r) {
                float v[kV];
#pragma unroll
                for (int i = 0; i < kV; ++i) v[i] = before[r].get(i);
                store_row_piece<T, kV>(final + sp.seq * state + r * (int64_t)p.dim, v);
            }
        }
        a = e;
    }
}

constexpr int kCvGradRows = 4;

template <typename T, int kW, int kV, bool kNear> __global__ __launch_bounds__(kBlock, 2) void cv_grad_kernel(const CvArgs p) {
    __shared__ float s_sum[kBlock * kV];
    uint32_t group;
    const CvPlace c = cv_place<kV>(p, group);
    const T *x = (const T *)p.x + (int64_t)c.b * p.x_b + c.d;
    T *dx = (T *)p.dx + (int64_t)c.b * p.tokens * p.dim + c.d;
    const int64_t state = (int64_t)(kW - 1) * p.dim;
    float w[kW][kV], bias[kV], dw[kW + 1][kV];
    cv_weights<T, kW, kV>(p, c.d, w, bias);
#pragma unroll
    for (int j = 0; j <= kW; ++j)
#pragma unroll
        for (int i = 0; i < kV; ++i) dw[j][i] = 0.0f;
    if (c.there && p.cu && p.dinitial)
        for (uint32_t i = c.strip; i < (uint32_t)p.n_seqs; i += p.strips)
            if (min(max(p.cu[i + 1], 0), p.tokens) <= min(max(p.cu[i], 0), p.tokens))
                for (int r = 0; r < kW - 1; ++r)
                    cv_copy_row<T, kV>(p.dfinal ? (const T *)p.dfinal + i * state + r * (int64_t)p.dim + c.d : nullptr, (T *)p.dinitial + i * state + r * (int64_t)p.dim + c.d);
    for (int a = c.t0; c.there && a < c.t1;) {
        const TsSpan sp = ts_span_at(p.cu, p.n_seqs, p.tokens, c.b, a);
        const int e = min(sp.hi, c.t1);
        if (sp.seq < 0) {
            for (int t = a; t < e; ++t) cv_copy_row<T, kV>(nullptr, dx + (int64_t)t * p.dim);
            a = e;
            continue;
        }
        float window[kW - 1][kV], g[kW - 1][kV];                     // inputs before token t, and g of the W - 1 before it
#pragma unroll
        for (int r = 0; r < kW - 1; ++r) {
            const RowPiece<T, kV> v = cv_line<T, kW, kV>(p, x, sp, c.d, a - kW + 1 + r);
#pragma unroll
            for (int i = 0; i < kV; ++i) {
                window[r][i] = v.get(i);
                g[r][i] = 0.0f;
            }
        }
        const int stop = e + kW - 1;                                 // the strip's last dx needs the W - 1 tokens behind it
        constexpr int kRows = kCvGradRows;
        const CvRow<T, kNear> x_row(p.x, p.x_t, c.b * p.x_b + a * p.x_t + c.d), d_row(p.dout, p.do_t, c.b * p.do_b + a * p.do_t + c.d),
            dx_row(p.dx, p.dim, ((int64_t)c.b * p.tokens + a) * p.dim + c.d);
        for (int i0 = 0; a + i0 < stop; i0 += kRows) {               // (as many tokens on in every lane)
            const int t = a + i0, last_row = min(sp.hi, stop) - 1 - a;
            RowPiece<T, kV> rows[kRows], ups[kRows];
            if (t + kRows <= e) {
#pragma unroll
                for (int k = 0; k < kRows; ++k) {
                    rows[k] = load_row_piece<T, kV>(x_row.at(i0 + k));
                    ups[k] = load_row_piece<T, kV>(d_row.at(i0 + k));
                }
            } else {
#pragma unroll
                for (int k = 0; k < kRows; ++k) {
                    rows[k] = load_row_piece<T, kV>(x_row.any(min(i0 + k, last_row)));
                    ups[k] = load_row_piece<T, kV>(d_row.any(min(i0 + k, last_row)));
                }
            }
            auto chunk = [&](auto all) {                             // all: its tokens are the strip's
                constexpr bool kAll = decltype(all)::value;
#pragma unroll
                for (int k = 0; k < kRows; ++k) {
                    const int now = t + k, to = now - kW + 1;        // the token that dx is found of
                    const bool own = kAll || now < e;
                    float d[kV];
#pragma unroll
                    for (int i = 0; i < kV; ++i) {
                        const float in = rows[k].get(i);
                        float y = fmaf(w[kW - 1][i], in, bias[i]), gt = ups[k].get(i);
#pragma unroll
                        for (int j = 0; j < kW - 1; ++j) y = fmaf(w[j][i], window[j][i], y);
                        if (p.silu) {
                            const float sig = ts_sigmoid(y);
                            gt *= sig * fmaf(y, 1.0f - sig, 1.0f);
                        }
                        if (!kAll) gt = now < sp.hi ? gt : 0.0f;
                        d[i] = kAll || now < sp.hi ? w[0][i] * gt : 0.0f;
#pragma unroll
                        for (int j = 1; j < kW; ++j)                 // (tokens that are not there: not even 0 times an infinite tap)
                            if (kAll || now - j < sp.hi) d[i] = fmaf(w[j][i], g[kW - 1 - j][i], d[i]);
#pragma unroll
                        for (int j = 0; j < kW - 1; ++j) dw[j][i] = own ? fmaf(gt, window[j][i], dw[j][i]) : dw[j][i];
                        dw[kW - 1][i] = own ? fmaf(gt, in, dw[kW - 1][i]) : dw[kW - 1][i];
                        dw[kW][i] = own ? dw[kW][i] + gt : dw[kW][i];
#pragma unroll
                        for (int j = 0; j < kW - 2; ++j) {
                            window[j][i] = window[j + 1][i];
                            g[j][i] = g[j + 1][i];
                        }
                        window[kW - 2][i] = in;
                        g[kW - 2][i] = gt;
                    }
                    if (kAll && to >= a) {                           // (before the tokens that a final state holds)
                        store_row_piece<T, kV>(const_cast<T *>(dx_row.at(i0 + k - kW + 1)), d);
                        continue;
                    }
                    if (now >= stop || (to < a && (a != sp.lo || !p.dinitial))) continue;
                    if (to < a) {                                    // a row of the state: of the first tokens' g alone, which are the newest
#pragma unroll
                        for (int i = 0; i < kV; ++i) {
                            d[i] = 0.0f;
#pragma unroll
                            for (int j = 0; j < kW - 1; ++j)
                                if (now - j >= a && now - j < sp.hi) d[i] = fmaf(w[j][i], g[kW - 2 - j][i], d[i]);
                        }
                    }
                    const int last = to - (sp.hi - kW + 1);          // its row of the final state, if it is there
                    if (p.dfinal && last >= 0) {
                        const RowPiece<T, kV> f = load_row_piece<T, kV>((const T *)p.dfinal + sp.seq * state + last * (int64_t)p.dim + c.d);
#pragma unroll
                        for (int i = 0; i < kV; ++i) d[i] += f.get(i);
                    }
                    store_row_piece<T, kV>(to >= sp.lo ? dx + (int64_t)to * p.dim : (T *)p.dinitial + sp.seq * state + (to - sp.lo + kW - 1) * (int64_t)p.dim + c.d, d);
                }
            };
            if (t + kRows <= e) chunk(std::true_type{});
            else chunk(std::false_type{});
        }
        a = e;
    }
    // the workgroup's strips' sums
    const int col = (int)threadIdx.x % p.cols, row = (int)threadIdx.x / p.cols, rows = kBlock / p.cols;
    const int piece = (int)(xcd_contiguous_id(blockIdx.x, gridDim.x) % (uint32_t)p.piece_blocks) * p.cols + col;
#pragma unroll
    for (int j = 0; j <= kW; ++j) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kV; ++i) s_sum[(row * kV + i) * p.cols + col] = dw[j][i];
        __syncthreads();
        if (row == 0 && piece < p.pieces) {
            float total[kV] = {};
            for (int r = 0; r < rows; ++r)
#pragma unroll
                for (int i = 0; i < kV; ++i) total[i] += s_sum[(r * kV + i) * p.cols + col];
            store_row_piece<float, kV>(p.sums + ((int64_t)group * (kW + 1) + j) * p.dim + c.d, total);
        }
    }
}

// The weights' gradients: sums over the workgroups' strips, 64 channels of one tap (or of the bias) to a workgroup
template <typename U> __global__ __launch_bounds__(kBlock) void cv_sum_kernel(const float *__restrict__ sums, U *dweight, U *dbias, int dim, int width, int64_t parts) {
    __shared__ float s_part[kBlock];
    const int d = (int)blockIdx.x * kWave + (int)threadIdx.x % kWave, j = (int)blockIdx.y, slice = (int)threadIdx.x / kWave;
    float total[4] = {0, 0, 0, 0};
    if (d < dim) {
        const float *from = sums + (int64_t)j * dim + d;
        const int64_t pitch = (int64_t)(width + 1) * dim;
        int64_t k = slice;
        for (; k + 12 < parts; k += 16)
#pragma unroll
            for (int e = 0; e < 4; ++e) total[e] += from[(k + 4 * e) * pitch];
        for (; k < parts; k += 4) total[0] += from[k * pitch];
    }
    s_part[threadIdx.x] = (total[0] + total[1]) + (total[2] + total[3]);
    __syncthreads();
    if (slice != 0 || d >= dim) return;
    const float all = (s_part[threadIdx.x] + s_part[threadIdx.x + 64]) + (s_part[threadIdx.x + 128] + s_part[threadIdx.x + 192]);
    if (j < width) {
        if (dweight) dweight[(int64_t)d * width + j] = from_f32<U>(all);
    } else if (dbias) {
        dbias[d] = from_f32<U>(all);
    }
}

// One token of each sequence: the state moves up by a row in place, so channels are no two threads'
template <typename T, int kW, int kV, int kRows> __global__ __launch_bounds__(kBlock) void cv_step_kernel(const CvArgs p, T *state, int64_t state_b, uint32_t blocks, int first) {
    const int64_t piece = (int64_t)(blockIdx.x % blocks) * kBlock + threadIdx.x;
    const int d = first + (int)piece * kV, b0 = (int)(blockIdx.x / blocks) * kRows;
    if (piece * kV + kV > p.dim - first) return;
    float w[kW][kV], bias[kV];
    RowPiece<T, kV> rows[kRows][kW];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
        const int64_t b = min(b0 + r, p.batch - 1);
#pragma unroll
        for (int j = 0; j < kW - 1; ++j) rows[r][j] = load_row_piece<T, kV>(state + b * state_b + (int64_t)j * p.dim + d);
        rows[r][kW - 1] = load_row_piece<T, kV>((const T *)p.x + b * p.x_b + d);
    }
    cv_weights<T, kW, kV>(p, d, w, bias);
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
        if (b0 + r >= p.batch) break;
        const int64_t b = b0 + r;
        float y[kV];
#pragma unroll
        for (int i = 0; i < kV; ++i) {
            y[i] = bias[i];
#pragma unroll
            for (int j = 0; j < kW; ++j) y[i] = fmaf(w[j][i], rows[r][j].get(i), y[i]);
            if (p.silu) y[i] *= ts_sigmoid(y[i]);
        }
        store_row_piece<T, kV>((T *)p.out + b * p.dim + d, y);
#pragma unroll
        for (int j = 0; j < kW - 1; ++j) {
            float v[kV];
#pragma unroll
            for (int i = 0; i < kV; ++i) v[i] = rows[r][j + 1].get(i);
            store_row_piece<T, kV>(state + b * state_b + (int64_t)j * p.dim + d, v);
        }
    }
}

template <typename T> __global__ __launch_bounds__(kBlock) void cv_copy_kernel(const T *from, T *to, int64_t n) {
    const int64_t i = (int64_t)blockIdx.x * kBlock + threadIdx.x;
    if (i < n) to[i] = from ? from[i] : from_f32<T>(0.0f);
}
template <typename T> static int cv_copy(const void *from, void *to, int64_t n, hipStream_t st) {
    if (!to || n == 0) return SS2D_OK;
    const int64_t wgs = (n + kBlock - 1) / kBlock;
    if (wgs > kTsLaunch / kBlock) return SS2D_ENOTSUP;
    cv_copy_kernel<T><<<(uint32_t)wgs, kBlock, 0, st>>>((const T *)from, (T *)to, n);
    return launch_status();
}

// ---- host ------------------------------------------------------------------------------------------------------------------------
static int cv_read(const ss2d_causal_conv_params *p, CvArgs &a) {
    a = {};
    if (!p || p->batch < 0 || p->seqlen < 0 || p->dim < 0 || p->n_seqs < 0) return SS2D_EINVAL;
    if (p->dtype < SS2D_F32 || p->dtype > SS2D_F16 || (p->weight_dtype != SS2D_F32 && p->weight_dtype != p->dtype)) return SS2D_EINVAL;
    if (p->cu_seqlens && (p->batch != 1 || p->n_seqs < 1)) return SS2D_EINVAL;
    if (p->width < 2 || p->width > 4 || p->seqlen > INT32_MAX - 256 || p->dim > 1 << 30) return SS2D_ENOTSUP;
    a.x = p->x; a.weight = p->weight; a.bias = p->bias; a.initial = p->initial_state; a.cu = p->cu_seqlens; a.out = p->out; a.final = p->final_state;
    a.x_b = p->x_batch_stride; a.x_t = p->x_token_stride;
    a.batch = p->batch; a.tokens = p->seqlen; a.dim = p->dim; a.n_seqs = p->cu_seqlens ? p->n_seqs : p->batch; a.silu = p->silu != 0;
    a.weight_f32 = p->weight_dtype == SS2D_F32 && p->dtype != SS2D_F32;
    return SS2D_OK;
}

// The grid for pieces of `v` channels: strips as long as they may be with enough threads, and `least` tokens at least (their ends are read twice).  -1: too many
static int64_t cv_grid(CvArgs &a, int v, int longest, int least, int64_t enough) {
    a.pieces = (int)(((int64_t)a.dim + v - 1) / v);
    a.cols = 1;
    while (a.cols < 64 && a.cols < a.pieces) a.cols *= 2;
    a.piece_blocks = (a.pieces + a.cols - 1) / a.cols;
    a.strip = longest;
    auto threads = [&] { return (int64_t)a.batch * ((a.tokens + a.strip - 1) / a.strip) * a.pieces; };
    while (a.strip > least && threads() < enough) a.strip /= 2;
    a.strips = (a.tokens + a.strip - 1) / a.strip;
    const int rows = kBlock / a.cols;
    const int64_t wgs = ((int64_t)a.batch * a.strips + rows - 1) / rows * a.piece_blocks;
    return wgs > kTsLaunch / kBlock ? -1 : wgs;
}
// The gradients' likewise: 37 tokens of 1024 channels, forward and gradients, 17.3 -> 11.9 us, 2 x 1024 of 2048 (2^22) 27.5 -> 25.0, 8 x 512 (2^23) 38.2 and 38.0,
// 8 x 4096 157 and 170 by two channels.  Strips: twice the threads take 8 x 2048 from 102 to 91 us, strips of 8 tokens, whose ends are read twice, 4 x 4096 of 1001 channels from 69 to 84.
static bool cv_few(const CvArgs &a) { return (int64_t)a.batch * a.tokens * a.dim <= kCvFew; }
static int cv_grad_vec(const CvArgs &a, int size) { return a.dim < 16 / size ? 1 : cv_few(a) ? 2 : 16 / size; }
// (the weights' sums take four threads a channel, which a launch counts in 32 bits)
static int64_t cv_grad_grid(CvArgs &a, int size) { return a.dim > kTsLaunch / kBlock * kWave ? -1 : cv_grid(a, cv_grad_vec(a, size), 64, cv_few(a) ? 8 : 16, 131072); }

// Offsets of a tensor of these strides, and of a dense one, are below 4 GB from the first row's (a row before it and chunks behind the last among them)
static bool cv_near(const CvArgs &a, int64_t size, int64_t batch, int64_t token) {
    constexpr int64_t kMost = 0xffffffff;
    if (batch < 0 || token < 0 || token > kMost / size || (a.batch > 1 && batch > kMost / size)) return false;
    const __int128 far = (__int128)(a.batch - 1) * batch + (__int128)(a.tokens + 64) * token + a.dim, dense = ((__int128)a.batch * a.tokens + 64) * a.dim;
    return far * size <= kMost && dense * size <= kMost;
}

// fn(T, width)
template <typename F> static int cv_with(int dtype, int width, F fn) {
    using std::integral_constant;
    auto typed = [&](auto t) {
        if (width == 2) return fn(t, integral_constant<int, 2>{});
        if (width == 3) return fn(t, integral_constant<int, 3>{});
        return fn(t, integral_constant<int, 4>{});
    };
    return dtype == SS2D_F32 ? typed(float{}) : dtype == SS2D_F16 ? typed(f16_t{}) : typed(bf16_t{});
}

}  // namespace ss2d

using namespace ss2d;

extern "C" int ss2d_causal_conv_fwd(const ss2d_causal_conv_params *params, void *stream) {
    CvArgs a;
    const int rc = cv_read(params, a);
    if (rc != SS2D_OK || a.dim == 0 || a.batch == 0) return rc;
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    return cv_with(params->dtype, params->width, [&](auto t, auto width) {
        using T = decltype(t);
        constexpr int kW = decltype(width)::value, kV = 16 / (int)sizeof(T);
        if (a.tokens == 0) return cv_copy<T>(a.initial, a.final, (int64_t)a.n_seqs * (kW - 1) * a.dim, st);
        if (!a.x || !a.weight || !a.out) return (int)SS2D_EINVAL;
        const bool few = cv_few(a);
        const int v = a.dim < kV ? 1 : few ? 2 : kV;
        const int64_t wgs = cv_grid(a, v, few ? kCvFewRows : 64, 4, few ? 262144 : 131072);
        if (wgs < 0) return (int)SS2D_ENOTSUP;
        a.near = cv_near(a, sizeof(T), a.x_b, a.x_t);
        if (v == 1) cv_kernel<T, kW, 1, false, kCvRows><<<(uint32_t)wgs, kBlock, 0, st>>>(a);
        else if (a.near && few) cv_kernel<T, kW, 2, true, kCvFewRows><<<(uint32_t)wgs, kBlock, 0, st>>>(a);
        else if (a.near) cv_kernel<T, kW, kV, true, kCvRows><<<(uint32_t)wgs, kBlock, 0, st>>>(a);
        else if (few) cv_kernel<T, kW, 2, false, kCvFewRows><<<(uint32_t)wgs, kBlock, 0, st>>>(a);
        else cv_kernel<T, kW, kV, false, kCvRows><<<(uint32_t)wgs, kBlock, 0, st>>>(a);
        return launch_status();
    });
}

extern "C" int64_t ss2d_causal_conv_bwd_workspace_bytes(const ss2d_causal_conv_bwd_params *params) {
    CvArgs a;
    const int rc = cv_read(params ? &params->fwd : nullptr, a);
    if (rc != SS2D_OK) return rc;
    if (a.dim == 0 || a.batch == 0 || a.tokens == 0) return 0;
    const int64_t wgs = cv_grad_grid(a, params->fwd.dtype == SS2D_F32 ? 4 : 2);
    return wgs < 0 ? (int64_t)SS2D_ENOTSUP : wgs / a.piece_blocks * (params->fwd.width + 1) * a.dim * 4;
}

extern "C" int ss2d_causal_conv_bwd(const ss2d_causal_conv_bwd_params *params, void *workspace, int64_t workspace_bytes, void *stream) {
    CvArgs a;
    const int rc = cv_read(params ? &params->fwd : nullptr, a);
    if (rc != SS2D_OK || a.dim == 0) return rc;
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    a.dout = params->dout; a.dfinal = params->dfinal_state; a.dx = params->dx; a.dinitial = params->dinitial_state;
    a.do_b = params->dout_batch_stride; a.do_t = params->dout_token_stride;
    const int width = params->fwd.width;
    return cv_with(params->fwd.dtype, width, [&](auto t, auto w) {
        using T = decltype(t);
        constexpr int kW = decltype(w)::value, kV = 16 / (int)sizeof(T);
        const bool wide = params->fwd.weight_dtype == SS2D_F32;
        if (a.batch == 0 || a.tokens == 0) {                         // no tokens: the weights' gradients are zeros, the state's what came in
            int status = wide ? cv_copy<float>(nullptr, params->dweight, (int64_t)a.dim * kW, st) : cv_copy<T>(nullptr, params->dweight, (int64_t)a.dim * kW, st);
            if (status == SS2D_OK) status = wide ? cv_copy<float>(nullptr, params->dbias, a.dim, st) : cv_copy<T>(nullptr, params->dbias, a.dim, st);
            return status != SS2D_OK ? status : cv_copy<T>(a.dfinal, a.dinitial, (int64_t)a.n_seqs * (kW - 1) * a.dim, st);
        }
        if (!a.x || !a.weight || !a.dout || !a.dx) return (int)SS2D_EINVAL;
        const int64_t wgs = cv_grad_grid(a, sizeof(T));
        if (wgs < 0) return (int)SS2D_ENOTSUP;
        const int64_t parts = wgs / a.piece_blocks;
        if (!workspace || reinterpret_cast<uintptr_t>(workspace) % 16) return (int)SS2D_EINVAL;
        if (workspace_bytes < parts * (kW + 1) * a.dim * 4) return (int)SS2D_ENOMEM;
        a.sums = (float *)workspace;
        a.near = cv_near(a, sizeof(T), a.x_b, a.x_t) && cv_near(a, sizeof(T), a.do_b, a.do_t);
        const int v = cv_grad_vec(a, sizeof(T));
        if (v == 1) cv_grad_kernel<T, kW, 1, false><<<(uint32_t)wgs, kBlock, 0, st>>>(a);
        else if (v == 2) a.near ? cv_grad_kernel<T, kW, 2, true><<<(uint32_t)wgs, kBlock, 0, st>>>(a) : cv_grad_kernel<T, kW, 2, false><<<(uint32_t)wgs, kBlock, 0, st>>>(a);
        else a.near ? cv_grad_kernel<T, kW, kV, true><<<(uint32_t)wgs, kBlock, 0, st>>>(a) : cv_grad_kernel<T, kW, kV, false><<<(uint32_t)wgs, kBlock, 0, st>>>(a);
        if (params->dweight || params->dbias) {
            const dim3 grid((a.dim + kWave - 1) / kWave, kW + 1);
            if (wide) cv_sum_kernel<float><<<grid, kBlock, 0, st>>>(a.sums, (float *)params->dweight, (float *)params->dbias, a.dim, kW, parts);
            else cv_sum_kernel<T><<<grid, kBlock, 0, st>>>(a.sums, (T *)params->dweight, (T *)params->dbias, a.dim, kW, parts);
        }
        return launch_status();
    });
}

extern "C" int ss2d_causal_conv_step(const ss2d_causal_conv_step_params *p, void *stream) {
    if (!p || p->batch < 0 || p->dim < 0) return SS2D_EINVAL;
    if (p->dtype < SS2D_F32 || p->dtype > SS2D_F16 || (p->weight_dtype != SS2D_F32 && p->weight_dtype != p->dtype)) return SS2D_EINVAL;
    if (p->width < 2 || p->width > 4 || p->dim > 1 << 30) return SS2D_ENOTSUP;
    if (p->batch == 0 || p->dim == 0) return SS2D_OK;
    if (!p->x || !p->weight || !p->state || !p->out) return SS2D_EINVAL;
    if (p->batch > 1 && p->state_batch_stride < (int64_t)(p->width - 1) * p->dim) return SS2D_EINVAL;
    CvArgs a = {};
    a.x = p->x; a.weight = p->weight; a.bias = p->bias; a.out = p->out; a.x_b = p->x_batch_stride; a.batch = p->batch; a.dim = p->dim; a.silu = p->silu != 0;
    a.weight_f32 = p->weight_dtype == SS2D_F32 && p->dtype != SS2D_F32;
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    return cv_with(p->dtype, p->width, [&](auto t, auto width) {
        using T = decltype(t);
        constexpr int kW = decltype(width)::value, kV = 16 / (int)sizeof(T), kRows = 4;
        const int whole = a.dim / kV, rest = a.dim % kV;
        auto go = [&](auto kernel, int pieces, int rows, int first) {
            const int64_t blocks = ((int64_t)pieces + kBlock - 1) / kBlock, wgs = blocks * (((int64_t)a.batch + rows - 1) / rows);
            if (wgs > kTsLaunch / kBlock) return (int)SS2D_ENOTSUP;
            kernel<<<(uint32_t)wgs, kBlock, 0, st>>>(a, (T *)p->state, p->state_batch_stride, (uint32_t)blocks, first);
            return launch_status();
        };
        // several sequences to a thread read the weights once, where there are threads enough (4096 channels, four sequences to a thread and one: 256 sequences, and 512, from where
        // on, 6.7 to 7.1 us either way; 1024 9.6 and 11.3)
        const bool many = (int64_t)a.batch * whole >= (1 << 18);
        int rc = whole == 0 ? SS2D_OK : many ? go(cv_step_kernel<T, kW, kV, kRows>, whole, kRows, 0) : go(cv_step_kernel<T, kW, kV, 1>, whole, 1, 0);
        if (rc == SS2D_OK && rest) rc = go(cv_step_kernel<T, kW, 1, 1>, rest, 1, whole * kV);      // (channels behind the last whole piece)
        return rc;
    });
}
