// Group norm of channel-last activations, with an activation behind it and their gradients: x (sample, position, channel), a group being cg neighbouring channels,
//     n = (x - mean) rstd,   y = act(n w + b),   mean and rstd = 1 / sqrt(var + eps) over a sample's positions and a group's channels.
// With d = dout act'(..) and m1, m2 the means over the group of d w and d w n:   dx = rstd (d w - m1 - n m2),   dw = sum d n,   db = sum d.
//
// Memory bounds it.  Two forms:
//   units   a sample's group is held in registers by a team of lanes -- part of a wavefront, or a workgroup -- and read once: tokens, and small maps in the
//           forward.  Gradients (one position): a team keeps its channels and walks over samples, with the weights' sums in registers.
//   slices  larger ones: a workgroup takes a slice of the positions for a bundle of whole groups (or a part of a wide one), channels side by side, so that rows are
//           read whole however narrow the groups; statistics first (each channel's running mean and squares about it, joined by rows, channels and slices:
//           no squares of what is not centred), then the values, which the caches still hold.
#include "row_piece.h"

namespace ss2d {

constexpr float kGnLog2e = 1.4426950408889634f;
constexpr int64_t kGnLaunch = 0xffffffff;                            // threads of a launch
constexpr int kGnPieces = 4;         // of a unit with a lane, at most

struct GnArgs {
    const void *x, *weight, *bias, *dout;
    void *out, *dx;
    float2 *stats;                   // [sample][group]: mean, rstd
    const float2 *read_stats;
    float *sums;                     // gradients: [part][d, d n][channel]
    float2 *means;                   // slices' gradients: [sample][group]: m1, m2
    float2 *parts;                   // slices' statistics: [sample][group][part of a wide group][slice]: mean, squares about it
    int64_t batch;
    int32_t positions, channels, groups, cg;
    float eps;
    int32_t silu, weight_f32;
    // units
    int32_t per_row;                 // pieces of a position's row of a group
    int32_t samples;                 // gradients: teams of a group, each with every samples-th sample
    // slices
    int32_t width, bundle_groups, bundles, group_parts;              // channels of a bundle; groups in it; bundles of a sample; parts of a group (1 where bundles hold whole ones)
    int32_t cols, slices, slice;     // pieces side by side; slices of a sample, positions of one
};

__device__ __forceinline__ float gn_sigmoid(float x) { return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-kGnLog2e * x)); }

template <typename T, int kV> __device__ __forceinline__ void gn_weights(const GnArgs &p, int c, float (&w)[kV], float (&b)[kV]) {
    auto read = [&](auto t) {
        using U = decltype(t);
#pragma unroll
        for (int i = 0; i < kV; ++i) { w[i] = 1.0f; b[i] = 0.0f; }
        if (p.weight) {
            const RowPiece<U, kV> r = load_row_piece<U, kV>((const U *)p.weight + c);
#pragma unroll
            for (int i = 0; i < kV; ++i) w[i] = r.get(i);
        }
        if (p.bias) {
            const RowPiece<U, kV> r = load_row_piece<U, kV>((const U *)p.bias + c);
#pragma unroll
            for (int i = 0; i < kV; ++i) b[i] = r.get(i);
        }
    };
    if (p.weight_f32) read(float{});
    else read(T{});
}

// v summed over a team of kLanes lanes (up to 64: neighbours in a wavefront; 256: the workgroup)
template <int kLanes> __device__ __forceinline__ float gn_team_sum(float v, float *s_team) {
#pragma unroll
    for (int over = 1; over < (kLanes < kWave ? kLanes : kWave); over *= 2) v += __shfl_xor(v, over, kWave);
    if constexpr (kLanes > kWave) {
        __syncthreads();
        if (threadIdx.x % kWave == 0) s_team[threadIdx.x / kWave] = v;
        __syncthreads();
        v = (s_team[0] + s_team[1]) + (s_team[2] + s_team[3]);
    }
    return v;
}

// ---- units ------------------------------------------------------------------------------------------------------------------------
template <typename T, int kV, int kLanes, int kK> __global__ __launch_bounds__(kBlock) void gn_unit_kernel(const GnArgs p) {
    __shared__ float s_team[4];
    constexpr int kTeams = kBlock / kLanes;
    const int64_t units = p.batch * p.groups, unit0 = (int64_t)blockIdx.x * kTeams + (int)threadIdx.x / kLanes, unit = unit0 < units ? unit0 : units - 1;
    const int lane = (int)threadIdx.x % kLanes, g = (int)(unit % p.groups), c0 = g * p.cg, pieces = p.per_row * p.positions;
    const int64_t row0 = unit / p.groups * p.positions;
    const T *x = (const T *)p.x + row0 * p.channels + c0;
    T *out = (T *)p.out + row0 * p.channels + c0;
    RowPiece<T, kV> rows[kK];
    int64_t at[kK];
    int col[kK], skip[kK];                                           // of a row's last piece, which ends with it, the values that the one before has
#pragma unroll
    for (int k = 0; k < kK; ++k) {
        const int q = min(lane + k * kLanes, pieces - 1), row = q / p.per_row, c = q % p.per_row * kV;
        col[k] = min(c, p.cg - kV);
        skip[k] = lane + k * kLanes < pieces ? c - col[k] : kV;
        at[k] = (int64_t)row * p.channels + col[k];
        rows[k] = load_row_piece<T, kV>(x + at[k]);
    }
    float sum = 0.0f;
#pragma unroll
    for (int k = 0; k < kK; ++k)
#pragma unroll
        for (int i = 0; i < kV; ++i) sum += i >= skip[k] ? rows[k].get(i) : 0.0f;
    const float count = (float)p.positions * (float)p.cg, mean = gn_team_sum<kLanes>(sum, s_team) / count;
    sum = 0.0f;
#pragma unroll
    for (int k = 0; k < kK; ++k)
#pragma unroll
        for (int i = 0; i < kV; ++i) {
            const float v = rows[k].get(i) - mean;
            sum = i >= skip[k] ? fmaf(v, v, sum) : sum;
        }
    const float rstd = 1.0f / sqrtf(gn_team_sum<kLanes>(sum, s_team) / count + p.eps);
    if (unit0 >= units) return;
    if (p.stats && lane == 0) p.stats[unit] = make_float2(mean, rstd);
#pragma unroll
    for (int k = 0; k < kK; ++k) {
        if (lane + k * kLanes >= pieces) break;
        float w[kV], b[kV], y[kV];
        gn_weights<T, kV>(p, c0 + col[k], w, b);
#pragma unroll
        for (int i = 0; i < kV; ++i) {
            y[i] = fmaf((rows[k].get(i) - mean) * rstd, w[i], b[i]);
            if (p.silu) y[i] *= gn_sigmoid(y[i]);
        }
        store_row_piece<T, kV>(out + at[k], y);
    }
}

// d = dout act'(n w + b)
__device__ __forceinline__ float gn_through(float dout, float n, float w, float b, int silu) {
    if (!silu) return dout;
    const float y = fmaf(n, w, b), sig = gn_sigmoid(y);
    return dout * (sig * fmaf(y, 1.0f - sig, 1.0f));
}

template <typename T, int kV, int kLanes, int kK> __global__ __launch_bounds__(kBlock) void gn_unit_grad_kernel(const GnArgs p) {
    __shared__ float s_team[4];
    constexpr int kTeams = kBlock / kLanes;
    const int64_t team0 = (int64_t)blockIdx.x * kTeams + (int)threadIdx.x / kLanes, teams = (int64_t)p.samples * p.groups, team = team0 < teams ? team0 : teams - 1;
    const int lane = (int)threadIdx.x % kLanes, g = (int)(team % p.groups), c0 = g * p.cg, first = (int)(team / p.groups);
    float w[kK][kV], b[kK][kV], dw[kK][kV], db[kK][kV];
    int col[kK], skip[kK];
#pragma unroll
    for (int k = 0; k < kK; ++k) {
        const int c = min(lane + k * kLanes, p.per_row - 1) * kV;
        col[k] = min(c, p.cg - kV);
        skip[k] = lane + k * kLanes < p.per_row ? c - col[k] : kV;
        gn_weights<T, kV>(p, c0 + col[k], w[k], b[k]);
#pragma unroll
        for (int i = 0; i < kV; ++i) dw[k][i] = db[k][i] = 0.0f;
    }
    const float share = 1.0f / (float)p.cg;
    RowPiece<T, kV> xs[kK], ds[kK];
    float2 stat;
    auto request = [&](int64_t n) {
        n = n < p.batch ? n : p.batch - 1;
#pragma unroll
        for (int k = 0; k < kK; ++k) {
            xs[k] = load_row_piece<T, kV>((const T *)p.x + n * p.channels + c0 + col[k]);
            ds[k] = load_row_piece<T, kV>((const T *)p.dout + n * p.channels + c0 + col[k]);
        }
        stat = p.read_stats[n * p.groups + g];
    };
    request(first);
    // (every team of a workgroup makes as many rounds, so that a workgroup's sums meet)
    const int64_t rounds = (p.batch + p.samples - 1) / p.samples;
    for (int64_t r = 0; r < rounds; ++r) {
        const int64_t n = first + r * p.samples;
        const bool in = n < p.batch && team0 < teams;
        float v[kK][kV], d[kK][kV], m1 = 0.0f, m2 = 0.0f;
        const float rstd = stat.y;
#pragma unroll
        for (int k = 0; k < kK; ++k)
#pragma unroll
            for (int i = 0; i < kV; ++i) {
                v[k][i] = (xs[k].get(i) - stat.x) * rstd;
                d[k][i] = gn_through(ds[k].get(i), v[k][i], w[k][i], b[k][i], p.silu);
                const bool own = i >= skip[k];
                m1 = own ? fmaf(d[k][i], w[k][i], m1) : m1;
                m2 = own ? fmaf(d[k][i] * w[k][i], v[k][i], m2) : m2;
                dw[k][i] = in ? fmaf(d[k][i], v[k][i], dw[k][i]) : dw[k][i];
                db[k][i] = in ? db[k][i] + d[k][i] : db[k][i];
            }
        if (r + 1 < rounds) request(n + p.samples);
        m1 = gn_team_sum<kLanes>(m1, s_team) * share;
        m2 = gn_team_sum<kLanes>(m2, s_team) * share;
        if (!in) continue;
#pragma unroll
        for (int k = 0; k < kK; ++k) {
            if (lane + k * kLanes >= p.per_row) break;
            float o[kV];
#pragma unroll
            for (int i = 0; i < kV; ++i) o[i] = rstd * (fmaf(d[k][i], w[k][i], -m1) - v[k][i] * m2);
            store_row_piece<T, kV>((T *)p.dx + n * p.channels + c0 + col[k], o);
        }
    }
    if (team0 >= teams || !p.sums) return;
#pragma unroll
    for (int k = 0; k < kK; ++k) {
        if (lane + k * kLanes >= p.per_row) break;
        float *to = p.sums + (int64_t)first * 2 * p.channels + c0 + col[k];
        store_row_piece<float, kV>(to, db[k]);
        store_row_piece<float, kV>(to + p.channels, dw[k]);
    }
}

// ---- slices -----------------------------------------------------------------------------------------------------------------------
struct GnPlace { int64_t n; int slice, bundle, g0, k, c0, width, begin, end, piece, row, rows, c; bool there; };

template <int kV> __device__ __forceinline__ GnPlace gn_place(const GnArgs &p) {
    GnPlace q;
    uint32_t id = xcd_contiguous_id(blockIdx.x, gridDim.x);
    q.bundle = (int)(id % (uint32_t)p.bundles); id /= (uint32_t)p.bundles;
    q.slice = (int)(id % (uint32_t)p.slices);
    q.n = id / (uint32_t)p.slices;
    if (p.group_parts > 1) {                                         // a part of one group
        const int part = q.bundle % p.group_parts;
        q.g0 = q.bundle / p.group_parts; q.k = 1;
        q.c0 = q.g0 * p.cg + part * p.width;
        q.width = min(p.width, p.cg - part * p.width);
    } else {
        q.g0 = q.bundle * p.bundle_groups; q.k = min(p.bundle_groups, p.groups - q.g0);
        q.c0 = q.g0 * p.cg; q.width = q.k * p.cg;
    }
    q.begin = q.slice * p.slice; q.end = min(q.begin + p.slice, p.positions);
    q.piece = (int)threadIdx.x % p.cols; q.row = (int)threadIdx.x / p.cols; q.rows = kBlock / p.cols;
    q.there = q.piece * kV < q.width;
    q.c = max(min(q.piece * kV, q.width - kV), 0);                   // inside the bundle
    return q;
}

constexpr int kGnRows = 8;           // rows of a chunk

// fn(team of lanes) for every group of the bundle: s_out[group] from entries by rows and channels
template <typename T, int kV> __global__ __launch_bounds__(kBlock) void gn_stats_kernel(const GnArgs p) {
    __shared__ float s_mean[kBlock * kV], s_square[kBlock * kV];
    const GnPlace q = gn_place<kV>(p);
    const int pitch = p.cols * kV;
    if (q.there) {
        const T *x = (const T *)p.x + q.n * p.positions * p.channels + q.c0 + q.c;
        float mean[kV] = {}, square[kV] = {}, count = 0.0f;
        for (int t = q.begin + q.row; t < q.end; t += kGnRows * q.rows) {
            RowPiece<T, kV> rows[kGnRows];
#pragma unroll
            for (int k = 0; k < kGnRows; ++k) rows[k] = load_row_piece<T, kV>(x + (int64_t)min(t + k * q.rows, q.end - 1) * p.channels);
#pragma unroll
            for (int k = 0; k < kGnRows; ++k) {
                if (t + k * q.rows >= q.end) break;
                count += 1.0f;
                const float share = __builtin_amdgcn_rcpf(count);
#pragma unroll
                for (int i = 0; i < kV; ++i) {
                    const float v = rows[k].get(i), off = v - mean[i];
                    mean[i] = fmaf(off, share, mean[i]);
                    square[i] = fmaf(off, v - mean[i], square[i]);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < kV; ++i) {
            s_mean[q.row * pitch + q.c + i] = mean[i];
            s_square[q.row * pitch + q.c + i] = square[i];
        }
    }
    __syncthreads();
    // a team of lanes to a group of the bundle: the entries of its rows and channels
    int lanes = kWave;
    while (lanes > 1 && lanes * q.k > kBlock) lanes /= 2;
    const int team = (int)threadIdx.x / lanes, lane = (int)threadIdx.x % lanes, len = q.end - q.begin, wide = p.group_parts > 1 ? q.width : p.cg;
    auto held = [&](int row) { return (float)((len - row + q.rows - 1) / q.rows); };       // positions of a row of threads (0: none)
    for (int j0 = 0; j0 < q.k; j0 += kBlock / lanes) {               // (as often for every lane)
        const int j = min(j0 + team, q.k - 1), entries = min(q.rows, len) * wide;
        float sum = 0.0f;
        for (int e = lane; e < entries; e += lanes) sum = fmaf(held(e / wide), s_mean[e / wide * pitch + j * wide + e % wide], sum);
        for (int over = 1; over < lanes; over *= 2) sum += __shfl_xor(sum, over, kWave);
        const float mean = sum / ((float)len * (float)wide);
        sum = 0.0f;
        for (int e = lane; e < entries; e += lanes) {
            const int from = e / wide * pitch + j * wide + e % wide;
            const float off = s_mean[from] - mean;
            sum += fmaf(held(e / wide) * off, off, s_square[from]);
        }
        for (int over = 1; over < lanes; over *= 2) sum += __shfl_xor(sum, over, kWave);
        if (lane == 0 && j0 + team < q.k) {
            const int part = p.group_parts > 1 ? q.bundle % p.group_parts : 0;
            p.parts[((q.n * p.groups + q.g0 + j) * p.group_parts + part) * p.slices + q.slice] = make_float2(mean, sum);
        }
    }
}

// A sample's group from its parts, by a team of lanes
__device__ __forceinline__ float2 gn_join(const GnArgs &p, int64_t unit, int lane, int lanes) {
    const int n = p.group_parts * p.slices;
    const float2 *from = p.parts + unit * n;
    auto held = [&](int e) {
        const int part = e / p.slices, s = e % p.slices, width = p.group_parts > 1 ? min(p.width, p.cg - part * p.width) : p.cg;
        return (float)min(p.slice, p.positions - s * p.slice) * (float)width;
    };
    const float count = (float)p.positions * (float)p.cg;
    float sum = 0.0f;
    for (int e = lane; e < n; e += lanes) sum = fmaf(held(e), from[e].x, sum);
    for (int over = 1; over < lanes; over *= 2) sum += __shfl_xor(sum, over, kWave);
    const float mean = sum / count;
    sum = 0.0f;
    for (int e = lane; e < n; e += lanes) {
        const float off = from[e].x - mean;
        sum += fmaf(held(e) * off, off, from[e].y);
    }
    for (int over = 1; over < lanes; over *= 2) sum += __shfl_xor(sum, over, kWave);
    return make_float2(mean, 1.0f / sqrtf(sum / count + p.eps));
}

constexpr int kGnMaxGroups = 512;    // of a bundle

template <typename T, int kV> __global__ __launch_bounds__(kBlock) void gn_apply_kernel(const GnArgs p) {
    __shared__ float2 s_stats[kGnMaxGroups];
    const GnPlace q = gn_place<kV>(p);
    int lanes = kWave;
    while (lanes > 1 && lanes * q.k > kBlock) lanes /= 2;
    const int team = (int)threadIdx.x / lanes, lane = (int)threadIdx.x % lanes;
    for (int j0 = 0; j0 < q.k; j0 += kBlock / lanes) {
        const int j = min(j0 + team, q.k - 1);
        const float2 s = gn_join(p, q.n * p.groups + q.g0 + j, lane, lanes);
        if (lane == 0) {
            s_stats[j] = s;
            if (p.stats && q.slice == 0) p.stats[q.n * p.groups + q.g0 + j] = s;
        }
    }
    __syncthreads();
    if (!q.there) return;
    const int64_t at = q.n * p.positions * p.channels + q.c0 + q.c;
    const T *x = (const T *)p.x + at;
    T *out = (T *)p.out + at;
    float w[kV], b[kV], mean[kV];
    gn_weights<T, kV>(p, q.c0 + q.c, w, b);
#pragma unroll
    for (int i = 0; i < kV; ++i) {
        const float2 s = s_stats[(q.c + i) / p.cg % q.k];            // (of a part of a group, its one)
        mean[i] = s.x;
        w[i] *= s.y;
    }
    for (int t = q.begin + q.row; t < q.end; t += kGnRows * q.rows) {
        RowPiece<T, kV> rows[kGnRows];
#pragma unroll
        for (int k = 0; k < kGnRows; ++k) rows[k] = load_row_piece<T, kV>(x + (int64_t)min(t + k * q.rows, q.end - 1) * p.channels);
#pragma unroll
        for (int k = 0; k < kGnRows; ++k) {
            if (t + k * q.rows >= q.end) break;
            float y[kV];
#pragma unroll
            for (int i = 0; i < kV; ++i) {
                y[i] = fmaf(rows[k].get(i) - mean[i], w[i], b[i]);
                if (p.silu) y[i] *= gn_sigmoid(y[i]);
            }
            store_row_piece<T, kV>(out + (int64_t)(t + k * q.rows) * p.channels, y);
        }
    }
}

// A slice's sums of d and d n for each channel (kSums), or its dx
template <typename T, int kV, bool kSums> __global__ __launch_bounds__(kBlock, 2) void gn_slice_grad_kernel(const GnArgs p) {
    __shared__ float s_d[kSums ? kBlock * kV : 1], s_dn[kSums ? kBlock * kV : 1];
    const GnPlace q = gn_place<kV>(p);
    const int pitch = p.cols * kV;
    if (q.there) {
        const int64_t at = q.n * p.positions * p.channels + q.c0 + q.c;
        const T *x = (const T *)p.x + at, *dout = (const T *)p.dout + at;
        T *dx = (T *)p.dx + at;
        float w[kV], b[kV], mean[kV], rstd[kV], m1[kV], m2[kV], d_sum[kV] = {}, dn_sum[kV] = {};
        gn_weights<T, kV>(p, q.c0 + q.c, w, b);
#pragma unroll
        for (int i = 0; i < kV; ++i) {
            const int64_t unit = q.n * p.groups + q.g0 + (q.c + i) / p.cg % q.k;
            const float2 s = p.read_stats[unit];
            mean[i] = s.x;
            rstd[i] = s.y;
            m1[i] = m2[i] = 0.0f;
            if constexpr (!kSums) {
                m1[i] = p.means[unit].x;
                m2[i] = p.means[unit].y;
            }
        }
        constexpr int kRows = kGnRows / 2;
        for (int t = q.begin + q.row; t < q.end; t += kRows * q.rows) {
            RowPiece<T, kV> xs[kRows], ds[kRows];
#pragma unroll
            for (int k = 0; k < kRows; ++k) {
                const int64_t from = (int64_t)min(t + k * q.rows, q.end - 1) * p.channels;
                xs[k] = load_row_piece<T, kV>(x + from);
                ds[k] = load_row_piece<T, kV>(dout + from);
            }
#pragma unroll
            for (int k = 0; k < kRows; ++k) {
                if (t + k * q.rows >= q.end) break;
                float o[kV];
#pragma unroll
                for (int i = 0; i < kV; ++i) {
                    const float n = (xs[k].get(i) - mean[i]) * rstd[i], d = gn_through(ds[k].get(i), n, w[i], b[i], p.silu);
                    if constexpr (kSums) {
                        d_sum[i] += d;
                        dn_sum[i] = fmaf(d, n, dn_sum[i]);
                    } else {
                        o[i] = rstd[i] * (fmaf(d, w[i], -m1[i]) - n * m2[i]);
                    }
                }
                if constexpr (!kSums) store_row_piece<T, kV>(dx + (int64_t)(t + k * q.rows) * p.channels, o);
            }
        }
        if constexpr (kSums) {
#pragma unroll
            for (int i = 0; i < kV; ++i) {
                s_d[q.row * pitch + q.c + i] = d_sum[i];
                s_dn[q.row * pitch + q.c + i] = dn_sum[i];
            }
        }
    }
    if constexpr (kSums) {
        __syncthreads();
        for (int c = threadIdx.x; c < q.width; c += kBlock) {
            float d = 0.0f, dn = 0.0f;
            for (int r = 0; r < q.rows; ++r) {
                d += s_d[r * pitch + c];
                dn += s_dn[r * pitch + c];
            }
            float *to = p.sums + (q.n * p.slices + q.slice) * 2 * p.channels + q.c0 + c;
            to[0] = d;
            to[p.channels] = dn;
        }
    }
}

// m1 and m2 of a sample's group, by a wavefront
template <typename T> __global__ __launch_bounds__(kBlock) void gn_means_kernel(const GnArgs p) {
    const int64_t unit = (int64_t)blockIdx.x * (kBlock / kWave) + (int)threadIdx.x / kWave;
    if (unit >= p.batch * p.groups) return;
    const int lane = (int)threadIdx.x % kWave, c0 = (int)(unit % p.groups) * p.cg;
    const float *from = p.sums + unit / p.groups * p.slices * 2 * p.channels + c0;
    float m1 = 0.0f, m2 = 0.0f;
    for (int64_t e = lane; e < (int64_t)p.slices * p.cg; e += kWave) {
        const int s = (int)(e / p.cg), c = (int)(e % p.cg);
        float w[1], b[1];
        gn_weights<T, 1>(p, c0 + c, w, b);
        m1 = fmaf(w[0], from[(int64_t)s * 2 * p.channels + c], m1);
        m2 = fmaf(w[0], from[(int64_t)s * 2 * p.channels + p.channels + c], m2);
    }
#pragma unroll
    for (int over = 1; over < kWave; over *= 2) {
        m1 += __shfl_xor(m1, over, kWave);
        m2 += __shfl_xor(m2, over, kWave);
    }
    const float count = (float)p.positions * (float)p.cg;
    if (lane == 0) p.means[unit] = make_float2(m1 / count, m2 / count);
}

// The weights' gradients: sums over the parts, 64 channels of db (y 0) or dw (1) to a workgroup of sixteen slices
template <typename U> __global__ __launch_bounds__(1024) void gn_sum_kernel(const float *__restrict__ sums, U *dweight, U *dbias, int channels, int64_t parts) {
    __shared__ float s_part[1024];
    const int c = (int)blockIdx.x * kWave + (int)threadIdx.x % kWave, slice = (int)threadIdx.x / kWave;
    U *to = blockIdx.y ? dweight : dbias;
    if (!to) return;
    float total[4] = {0, 0, 0, 0};
    if (c < channels) {
        const float *from = sums + (int64_t)blockIdx.y * channels + c;
        const int64_t pitch = 2 * (int64_t)channels;
        int64_t k = slice;
        for (; k + 48 < parts; k += 64)
#pragma unroll
            for (int e = 0; e < 4; ++e) total[e] += from[(k + 16 * e) * pitch];
        for (; k < parts; k += 16) total[0] += from[k * pitch];
    }
    s_part[threadIdx.x] = (total[0] + total[1]) + (total[2] + total[3]);
    __syncthreads();
    if (slice != 0 || c >= channels) return;
    float all = 0.0f;
#pragma unroll
    for (int s = 0; s < 16; ++s) all += s_part[s * kWave + threadIdx.x];
    to[c] = from_f32<U>(all);
}

template <typename U> __global__ __launch_bounds__(kBlock) void gn_clear_kernel(U *to, int n) {
    const int i = (int)blockIdx.x * kBlock + (int)threadIdx.x;
    if (i < n) to[i] = from_f32<U>(0.0f);
}

// ---- host ------------------------------------------------------------------------------------------------------------------------
static int gn_read(const ss2d_group_norm_params *p, GnArgs &a) {
    a = {};
    if (!p || p->batch < 0 || p->positions < 0 || p->channels < 1 || p->groups < 1 || p->channels % p->groups) return SS2D_EINVAL;
    if (p->dtype < SS2D_F32 || p->dtype > SS2D_F16 || (p->weight_dtype != SS2D_F32 && p->weight_dtype != p->dtype)) return SS2D_EINVAL;
    if (p->batch > INT32_MAX || p->positions > INT32_MAX - 65536 || p->channels > (1 << 30)) return SS2D_ENOTSUP;
    a.x = p->x; a.weight = p->weight; a.bias = p->bias; a.out = p->out; a.stats = (float2 *)p->stats; a.batch = p->batch;
    a.positions = (int)p->positions; a.channels = p->channels; a.groups = p->groups; a.cg = p->channels / p->groups; a.eps = p->eps; a.silu = p->silu != 0;
    a.weight_f32 = p->weight_dtype == SS2D_F32 && p->dtype != SS2D_F32;
    return SS2D_OK;
}

// Values to a piece: 16 bytes' worth, or less where a group is narrower
static int gn_vec(int cg, int size) {
    int v = 16 / size;
    while (v > cg) v /= 2;
    return v;
}

// Lanes of a team and pieces with a lane of it; false: the unit does not fit
static bool gn_unit(GnArgs &a, int v, int &lanes, int &each) {
    a.per_row = (a.cg + v - 1) / v;
    const int64_t pieces = (int64_t)a.per_row * a.positions;
    if (pieces > kBlock * kGnPieces) return false;
    if (pieces <= kWave * kGnPieces) {
        lanes = 1;
        while (lanes < kWave && lanes < pieces) lanes *= 2;
    } else {
        lanes = kBlock;
    }
    each = 1;
    while (each * lanes < pieces) each *= 2;
    return true;
}

static bool gn_slices(GnArgs &a, int size) {
    const int v = a.cg * (int64_t)a.groups < 16 / size ? 1 : 16 / size, most = kWave * v;
    if (a.cg > most) {
        a.bundle_groups = 1; a.width = most;
        a.group_parts = (a.cg + most - 1) / most;
        a.width = (a.cg + a.group_parts - 1) / a.group_parts;
        while (a.cg % a.width && a.cg % a.width < v) a.width -= 1;   // (no part narrower than a piece)
        a.group_parts = (a.cg + a.width - 1) / a.width;
        a.bundles = a.groups * a.group_parts;
    } else {
        a.group_parts = 1;
        a.bundle_groups = most / a.cg < a.groups ? most / a.cg : a.groups;
        a.width = a.bundle_groups * a.cg;
        a.bundles = (a.groups + a.bundle_groups - 1) / a.bundle_groups;
        // the last bundle has a piece at least too
        while (a.bundles > 1 && (a.groups - (a.bundles - 1) * a.bundle_groups) * a.cg < v) {
            a.bundle_groups -= 1;
            a.width = a.bundle_groups * a.cg;
            a.bundles = (a.groups + a.bundle_groups - 1) / a.bundle_groups;
        }
    }
    const int pieces = (a.width + v - 1) / v;
    a.cols = 1;
    while (a.cols < pieces) a.cols *= 2;
    const int rows = kBlock / a.cols;
    const int64_t others = a.batch * a.bundles, enough = 2048, most_slices = (a.positions + (int64_t)rows * 4 - 1) / (rows * 4);
    int64_t n = (enough + others - 1) / (others > 0 ? others : 1);
    n = n < most_slices ? n : most_slices;
    n = n < 1 ? 1 : n;
    a.slice = (int)((a.positions + n - 1) / n);
    a.slices = (int)((a.positions + (int64_t)a.slice - 1) / a.slice);
    return others * a.slices <= kGnLaunch / kBlock;
}

// fn(T, pieces' values, lanes, each) of a team
template <typename F> static int gn_team(int dtype, int v, int lanes, int each, F fn) {
    using std::integral_constant;
    auto by_each = [&](auto t, auto vec, auto l) {
        if constexpr (decltype(l)::value < kWave) return fn(t, vec, l, integral_constant<int, 1>{});
        else if (each == 1) return fn(t, vec, l, integral_constant<int, 1>{});
        else if (each == 2) return fn(t, vec, l, integral_constant<int, 2>{});
        else return fn(t, vec, l, integral_constant<int, 4>{});
    };
    auto by_lanes = [&](auto t, auto vec) {
        switch (lanes) {
        case 1: return by_each(t, vec, integral_constant<int, 1>{});
        case 2: return by_each(t, vec, integral_constant<int, 2>{});
        case 4: return by_each(t, vec, integral_constant<int, 4>{});
        case 8: return by_each(t, vec, integral_constant<int, 8>{});
        case 16: return by_each(t, vec, integral_constant<int, 16>{});
        case 32: return by_each(t, vec, integral_constant<int, 32>{});
        case 64: return by_each(t, vec, integral_constant<int, 64>{});
        default: return by_each(t, vec, integral_constant<int, 256>{});
        }
    };
    auto by_vec = [&](auto t) {
        if constexpr (sizeof(t) == 2)
            if (v == 8) return by_lanes(t, integral_constant<int, 8>{});
        if (v == 4) return by_lanes(t, integral_constant<int, 4>{});
        return v == 2 ? by_lanes(t, integral_constant<int, 2>{}) : by_lanes(t, integral_constant<int, 1>{});
    };
    return dtype == SS2D_F32 ? by_vec(float{}) : dtype == SS2D_F16 ? by_vec(f16_t{}) : by_vec(bf16_t{});
}

// fn(T, pieces' values) of a slice
template <typename F> static int gn_sliced(int dtype, int channels, F fn) {
    using std::integral_constant;
    auto by_vec = [&](auto t) {
        constexpr int kV = 16 / (int)sizeof(t);
        return channels < kV ? fn(t, integral_constant<int, 1>{}) : fn(t, integral_constant<int, kV>{});
    };
    return dtype == SS2D_F32 ? by_vec(float{}) : dtype == SS2D_F16 ? by_vec(f16_t{}) : by_vec(bf16_t{});
}

static int gn_size(int dtype) { return dtype == SS2D_F32 ? 4 : 2; }

// Teams of a group that walk over the samples
static int gn_samples(const GnArgs &a, int lanes) {
    const int64_t wanted = 2048 * kWave / ((int64_t)lanes * a.groups);
    return (int)(wanted < 1 ? 1 : wanted < a.batch ? wanted : a.batch);
}

}  // namespace ss2d

using namespace ss2d;

extern "C" int64_t ss2d_group_norm_workspace_bytes(const ss2d_group_norm_params *params) {
    GnArgs a;
    const int rc = gn_read(params, a);
    if (rc != SS2D_OK) return rc;
    int lanes, each;
    if (a.batch == 0 || a.positions == 0 || gn_unit(a, gn_vec(a.cg, gn_size(params->dtype)), lanes, each)) return 0;
    if (!gn_slices(a, gn_size(params->dtype))) return SS2D_ENOTSUP;
    return a.batch * a.groups * a.group_parts * a.slices * 8;
}

extern "C" int ss2d_group_norm_fwd(const ss2d_group_norm_params *params, void *workspace, int64_t workspace_bytes, void *stream) {
    GnArgs a;
    const int rc = gn_read(params, a);
    if (rc != SS2D_OK || a.batch == 0 || a.positions == 0) return rc;
    if (!a.x || !a.out) return SS2D_EINVAL;
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    const int size = gn_size(params->dtype), v = gn_vec(a.cg, size);
    int lanes, each;
    if (gn_unit(a, v, lanes, each))
        return gn_team(params->dtype, v, lanes, each, [&](auto t, auto vec, auto l, auto k) {
            constexpr int kLanes = decltype(l)::value, kTeams = kBlock / kLanes;
            const int64_t wgs = (a.batch * a.groups + kTeams - 1) / kTeams;
            if (wgs > kGnLaunch / kBlock) return (int)SS2D_ENOTSUP;
            gn_unit_kernel<decltype(t), decltype(vec)::value, kLanes, decltype(k)::value><<<(uint32_t)wgs, kBlock, 0, st>>>(a);
            return launch_status();
        });
    if (!gn_slices(a, size)) return SS2D_ENOTSUP;
    if (!workspace || reinterpret_cast<uintptr_t>(workspace) % 16) return SS2D_EINVAL;
    if (workspace_bytes < a.batch * a.groups * a.group_parts * a.slices * 8) return SS2D_ENOMEM;
    a.parts = (float2 *)workspace;
    return gn_sliced(params->dtype, a.channels, [&](auto t, auto vec) {
        const uint32_t wgs = (uint32_t)(a.batch * a.bundles * a.slices);
        gn_stats_kernel<decltype(t), decltype(vec)::value><<<wgs, kBlock, 0, st>>>(a);
        gn_apply_kernel<decltype(t), decltype(vec)::value><<<wgs, kBlock, 0, st>>>(a);
        return launch_status();
    });
}

static int64_t gn_bwd_plan(const ss2d_group_norm_params *p, GnArgs &a, int &lanes, int &each) {
    const int v = gn_vec(a.cg, gn_size(p->dtype));
    if (a.positions == 1 && gn_unit(a, v, lanes, each)) {
        a.samples = gn_samples(a, lanes);
        return (int64_t)a.samples * 2 * a.channels * 4;
    }
    lanes = 0;
    if (!gn_slices(a, gn_size(p->dtype))) return SS2D_ENOTSUP;
    return (a.batch * a.slices * 2 * a.channels * 4 + 15) / 16 * 16 + a.batch * a.groups * 8;
}

extern "C" int64_t ss2d_group_norm_bwd_workspace_bytes(const ss2d_group_norm_bwd_params *params) {
    GnArgs a;
    const int rc = gn_read(params ? &params->fwd : nullptr, a);
    if (rc != SS2D_OK) return rc;
    int lanes, each;
    return a.batch == 0 || a.positions == 0 ? 0 : gn_bwd_plan(&params->fwd, a, lanes, each);
}

extern "C" int ss2d_group_norm_bwd(const ss2d_group_norm_bwd_params *params, void *workspace, int64_t workspace_bytes, void *stream) {
    GnArgs a;
    const int rc = gn_read(params ? &params->fwd : nullptr, a);
    if (rc != SS2D_OK) return rc;
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    const int dtype = params->fwd.dtype;
    const bool wide = params->fwd.weight_dtype == SS2D_F32;
    auto weights = [&](auto fn) {                                    // fn of a weight's type
        if (wide) fn(float{});
        else if (dtype == SS2D_F16) fn(f16_t{});
        else fn(bf16_t{});
    };
    if (a.batch == 0 || a.positions == 0) {
        weights([&](auto u) {
            using U = decltype(u);
            for (void *to : {params->dweight, params->dbias})
                if (to) gn_clear_kernel<U><<<(a.channels + kBlock - 1) / kBlock, kBlock, 0, st>>>((U *)to, a.channels);
        });
        return launch_status();
    }
    a.dout = params->dout; a.dx = params->dx; a.read_stats = (const float2 *)params->fwd.stats;
    if (!a.x || !a.dout || !a.dx || !a.read_stats) return SS2D_EINVAL;
    int lanes, each;
    const int64_t need = gn_bwd_plan(&params->fwd, a, lanes, each);
    if (need < 0) return (int)need;
    if (!workspace || reinterpret_cast<uintptr_t>(workspace) % 16) return SS2D_EINVAL;
    if (workspace_bytes < need) return SS2D_ENOMEM;
    a.sums = (float *)workspace;
    int status;
    int64_t parts;
    if (lanes) {
        parts = a.samples;
        status = gn_team(dtype, gn_vec(a.cg, gn_size(dtype)), lanes, each, [&](auto t, auto vec, auto l, auto k) {
            constexpr int kLanes = decltype(l)::value, kTeams = kBlock / kLanes;
            const int64_t wgs = ((int64_t)a.samples * a.groups + kTeams - 1) / kTeams;
            if (wgs > kGnLaunch / kBlock) return (int)SS2D_ENOTSUP;
            gn_unit_grad_kernel<decltype(t), decltype(vec)::value, kLanes, decltype(k)::value><<<(uint32_t)wgs, kBlock, 0, st>>>(a);
            return launch_status();
        });
    } else {
        parts = a.batch * a.slices;
        a.means = (float2 *)((uint8_t *)workspace + (parts * 2 * a.channels * 4 + 15) / 16 * 16);
        const int64_t teams = (a.batch * a.groups + kBlock / kWave - 1) / (kBlock / kWave);
        if (teams > kGnLaunch / kBlock) return SS2D_ENOTSUP;
        status = gn_sliced(dtype, a.channels, [&](auto t, auto vec) {
            const uint32_t wgs = (uint32_t)(a.batch * a.bundles * a.slices);
            gn_slice_grad_kernel<decltype(t), decltype(vec)::value, true><<<wgs, kBlock, 0, st>>>(a);
            gn_means_kernel<decltype(t)><<<(uint32_t)teams, kBlock, 0, st>>>(a);
            gn_slice_grad_kernel<decltype(t), decltype(vec)::value, false><<<wgs, kBlock, 0, st>>>(a);
            return launch_status();
        });
    }
    if (status != SS2D_OK || (!params->dweight && !params->dbias)) return status;
    weights([&](auto u) {
        using U = decltype(u);
        gn_sum_kernel<U><<<dim3((a.channels + kWave - 1) / kWave, 2), 1024, 0, st>>>(a.sums, (U *)params->dweight, (U *)params->dbias, a.channels, parts);
    });
    return launch_status();
}
