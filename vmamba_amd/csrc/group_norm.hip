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
// 8192 rows of 2048 channels, 16 groups, bf16: 16 us, gradients 20 (5 TB/s) and 6 for the weights' sums.  32 maps of 56 x 56 x 192, 32 groups, fp16: statistics 10.5 and
// values 15.5 us, of one chunk of rows to each of 1280 workgroups: a launch, one latency and the copy's time each (7 and 10).
#include "row_piece.h"

namespace ss2d {

constexpr float kGnLog2e = 1.4426950408889634f;
constexpr int64_t kGnLaunch = 0xffffffff;                            // threads of a launch
constexpr int64_t kGnThreads = 262144;   // of the teams that walk over samples: four wavefronts to a SIMD
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
    int32_t samples;                 // teams of a group, each with every samples-th sample
    // slices
    int32_t width, bundle_groups, bundles, group_parts;              // channels of a bundle; groups in it; bundles of a sample; parts of a group (1 where bundles hold whole ones)
    int32_t cols, slices, slice;     // pieces side by side; slices of a sample, positions of one
    int32_t part_slices, part_slice; // those of the statistics
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

// v summed over a team of kLanes lanes (up to 64: neighbours in a wavefront; 256: the workgroup), left with all of them.  Inside a row of 16 lanes by
// additions that take their operand from another lane: neighbours, pairs, then mirrored halves and rows (whose quads and halves are of one value by then).
__device__ __forceinline__ float gn_swapped16(float v) {
    const auto r = __builtin_amdgcn_permlane16_swap(f32_to_bits(v), f32_to_bits(v), false, false);
    return bits_to_f32(r[0]) + bits_to_f32(r[1]);
}
__device__ __forceinline__ float gn_swapped32(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(f32_to_bits(v), f32_to_bits(v), false, false);
    return bits_to_f32(r[0]) + bits_to_f32(r[1]);
}
template <int kLanes> __device__ __forceinline__ float gn_team_sum(float v, float *s_team) {
    if constexpr (kLanes >= 2) v += dpp_move<0xB1>(0.0f, v);
    if constexpr (kLanes >= 4) v += dpp_move<0x4E>(0.0f, v);
    if constexpr (kLanes >= 8) v += dpp_move<0x141>(0.0f, v);
    if constexpr (kLanes >= 16) v += dpp_move<0x140>(0.0f, v);
    if constexpr (kLanes >= 32) v = gn_swapped16(v);
    if constexpr (kLanes >= 64) v = gn_swapped32(v);
    if constexpr (kLanes > kWave) {
        __syncthreads();
        if (threadIdx.x % kWave == 0) s_team[threadIdx.x / kWave] = v;
        __syncthreads();
        v = (s_team[0] + s_team[1]) + (s_team[2] + s_team[3]);
    }
    return v;
}

// ---- units ------------------------------------------------------------------------------------------------------------------------
// A team has a group, and every samples-th sample's: the next one's loads are on their way while one is worked on (8192 rows of 2048 channels, 16 groups: 16 us, 4.2 TB/s;
// 131072 rows: 194, 5.5 TB/s.  Each team's four units asked for at once and the workgroup done with them: 17.6 and 215).
template <typename T, int kV, int kLanes, int kK> __global__ __launch_bounds__(kBlock) void gn_unit_kernel(const GnArgs p) {
    __shared__ float s_team[4];
    constexpr int kTeams = kBlock / kLanes;
    const uint32_t teams = (uint32_t)p.samples * (uint32_t)p.groups, team0 = blockIdx.x * (uint32_t)kTeams + threadIdx.x / kLanes, team = min(team0, teams - 1);
    const int lane = (int)threadIdx.x % kLanes, g = (int)(team % (uint32_t)p.groups), first = (int)(team / (uint32_t)p.groups), c0 = g * p.cg, pieces = p.per_row * p.positions;
    const int64_t pitch = (int64_t)p.positions * p.channels;
    RowPiece<T, kV> rows[kK];
    int64_t at[kK];
    int col[kK], skip[kK];                                           // of a row's last piece, which ends with it, the values that the one before has
#pragma unroll
    for (int k = 0; k < kK; ++k) {
        const int q = min(lane + k * kLanes, pieces - 1), row = p.positions == 1 ? 0 : q / p.per_row, c = (q - row * p.per_row) * kV;
        col[k] = min(c, p.cg - kV);
        skip[k] = lane + k * kLanes < pieces ? c - col[k] : kV;
        at[k] = (int64_t)row * p.channels + c0 + col[k];
    }
    auto request = [&](int64_t n) {
#pragma unroll
        for (int k = 0; k < kK; ++k) rows[k] = load_row_piece<T, kV>((const T *)p.x + min(n, p.batch - 1) * pitch + at[k]);
    };
    request(first);
    float w[kK][kV], b[kK][kV];
#pragma unroll
    for (int k = 0; k < kK; ++k) gn_weights<T, kV>(p, c0 + col[k], w[k], b[k]);
    const float share = 1.0f / ((float)p.positions * (float)p.cg);
    const bool ragged = p.cg % kV != 0;                              // (uniform)
    const int64_t rounds = (p.batch + p.samples - 1) / p.samples;
    for (int64_t r = 0; r < rounds; ++r) {                           // (as many for every team, so that a workgroup's sums meet)
        const int64_t n = first + r * p.samples;
        float v[kK][kV];
#pragma unroll
        for (int k = 0; k < kK; ++k)
#pragma unroll
            for (int i = 0; i < kV; ++i) v[k][i] = rows[k].get(i);
        if (r + 1 < rounds) request(n + p.samples);
        float sum = 0.0f;
#pragma unroll
        for (int k = 0; k < kK; ++k) {
            float part = 0.0f;
            if (ragged) {
#pragma unroll
                for (int i = 0; i < kV; ++i) part += i >= skip[k] ? v[k][i] : 0.0f;
            } else {
#pragma unroll
                for (int i = 0; i < kV; ++i) part += v[k][i];
                part = skip[k] ? 0.0f : part;
            }
            sum += part;
        }
        const float mean = gn_team_sum<kLanes>(sum, s_team) * share;
        sum = 0.0f;
#pragma unroll
        for (int k = 0; k < kK; ++k) {
            float part = 0.0f;
#pragma unroll
            for (int i = 0; i < kV; ++i) {
                v[k][i] -= mean;
                part = !ragged || i >= skip[k] ? fmaf(v[k][i], v[k][i], part) : part;
            }
            sum += skip[k] < kV ? part : 0.0f;
        }
        const float rstd = __builtin_amdgcn_rsqf(fmaf(gn_team_sum<kLanes>(sum, s_team), share, p.eps));
        if (n >= p.batch || team0 >= teams) continue;
        if (p.stats && lane == 0) p.stats[n * p.groups + g] = make_float2(mean, rstd);
        T *to = (T *)p.out + n * pitch;
#pragma unroll
        for (int k = 0; k < kK; ++k) {
            if (lane + k * kLanes >= pieces) break;
            float y[kV];
#pragma unroll
            for (int i = 0; i < kV; ++i) {
                y[i] = fmaf(v[k][i] * rstd, w[k][i], b[k][i]);
                if (p.silu) y[i] *= gn_sigmoid(y[i]);
            }
            store_row_piece<T, kV>(to + at[k], y);
        }
    }
}

// d = dout act'(n w + b)
__device__ __forceinline__ float gn_through(float dout, float n, float w, float b, int silu) {
    if (!silu) return dout;
    const float y = fmaf(n, w, b), sig = gn_sigmoid(y);
    return dout * (sig * fmaf(y, 1.0f - sig, 1.0f));
}

template <typename T, int kV, int kLanes, int kK, int kUnits> __global__ __launch_bounds__(kBlock) void gn_unit_grad_kernel(const GnArgs p) {
    __shared__ float s_team[4];
    constexpr int kTeams = kBlock / kLanes;
    const uint32_t teams = (uint32_t)p.samples * (uint32_t)p.groups, team0 = blockIdx.x * (uint32_t)kTeams + threadIdx.x / kLanes, team = min(team0, teams - 1);
    const int lane = (int)threadIdx.x % kLanes, g = (int)(team % (uint32_t)p.groups), first = (int)(team / (uint32_t)p.groups), c0 = g * p.cg;
    float w[kK][kV], b[kK][kV], dw[kK][kV], db[kK][kV];
    int col[kK], skip[kK];
#pragma unroll
    for (int k = 0; k < kK; ++k) {
        const int c = min(lane + k * kLanes, p.per_row - 1) * kV;
        col[k] = c0 + min(c, p.cg - kV);
        skip[k] = lane + k * kLanes < p.per_row ? c0 + c - col[k] : kV;
        gn_weights<T, kV>(p, col[k], w[k], b[k]);
#pragma unroll
        for (int i = 0; i < kV; ++i) dw[k][i] = db[k][i] = 0.0f;
    }
    const float share = 1.0f / (float)p.cg;
    RowPiece<T, kV> xs[kUnits][kK], ds[kUnits][kK];
    float2 stat[kUnits];
    auto sample = [&](int64_t r, int u) { return (int64_t)first + (r * kUnits + u) * p.samples; };
    auto request = [&](int64_t r) {
#pragma unroll
        for (int u = 0; u < kUnits; ++u) {
            const int64_t n = min(sample(r, u), p.batch - 1);
#pragma unroll
            for (int k = 0; k < kK; ++k) {
                xs[u][k] = load_row_piece<T, kV>((const T *)p.x + n * p.channels + col[k]);
                ds[u][k] = load_row_piece<T, kV>((const T *)p.dout + n * p.channels + col[k]);
            }
            stat[u] = p.read_stats[n * p.groups + g];
        }
    };
    request(0);
    // (every team of a workgroup makes as many rounds, so that a workgroup's sums meet)
    const int64_t rounds = (p.batch + (int64_t)p.samples * kUnits - 1) / ((int64_t)p.samples * kUnits);
    for (int64_t r = 0; r < rounds; ++r) {
        float v[kUnits][kK][kV], d[kUnits][kK][kV], m1[kUnits], m2[kUnits], rstd[kUnits];
#pragma unroll
        for (int u = 0; u < kUnits; ++u) {
            const bool in = sample(r, u) < p.batch;
            m1[u] = m2[u] = 0.0f;
            rstd[u] = stat[u].y;
#pragma unroll
            for (int k = 0; k < kK; ++k)
#pragma unroll
                for (int i = 0; i < kV; ++i) {
                    v[u][k][i] = (xs[u][k].get(i) - stat[u].x) * rstd[u];
                    d[u][k][i] = in ? gn_through(ds[u][k].get(i), v[u][k][i], w[k][i], b[k][i], p.silu) : 0.0f;
                    const float dn = d[u][k][i] * w[k][i];
                    const bool own = i >= skip[k];
                    m1[u] += own ? dn : 0.0f;
                    m2[u] = own ? fmaf(dn, v[u][k][i], m2[u]) : m2[u];
                    dw[k][i] = in ? fmaf(d[u][k][i], v[u][k][i], dw[k][i]) : dw[k][i];
                    db[k][i] += d[u][k][i];
                }
        }
        if (r + 1 < rounds) request(r + 1);
#pragma unroll
        for (int u = 0; u < kUnits; ++u) {
            m1[u] = gn_team_sum<kLanes>(m1[u], s_team) * share;
            m2[u] = gn_team_sum<kLanes>(m2[u], s_team) * share;
            if (sample(r, u) >= p.batch || team0 >= teams) continue;
#pragma unroll
            for (int k = 0; k < kK; ++k) {
                if (lane + k * kLanes >= p.per_row) break;
                float o[kV];
#pragma unroll
                for (int i = 0; i < kV; ++i) o[i] = rstd[u] * (fmaf(d[u][k][i], w[k][i], -m1[u]) - v[u][k][i] * m2[u]);
                store_row_piece<T, kV>((T *)p.dx + sample(r, u) * p.channels + col[k], o);
            }
        }
    }
    if (team0 >= teams || !p.sums) return;
#pragma unroll
    for (int k = 0; k < kK; ++k) {
        if (lane + k * kLanes >= p.per_row) break;
        float *to = p.sums + (int64_t)first * 2 * p.channels + col[k];
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
    q.begin = q.slice * p.slice; q.end = q.begin + min(p.slice, p.positions - q.begin);
    q.piece = (int)threadIdx.x % p.cols; q.row = (int)threadIdx.x / p.cols; q.rows = kBlock / p.cols;
    q.there = q.piece * kV < q.width && q.row < q.rows;
    q.c = max(min(q.piece * kV, q.width - kV), 0);                   // inside the bundle
    return q;
}

// fn(i, group of the bundle) for the channels of a lane's piece
template <int kV, typename F> __device__ __forceinline__ void gn_by_group(const GnArgs &p, const GnPlace &q, F fn) {
    int g = p.group_parts > 1 ? 0 : q.c / p.cg, left = p.group_parts > 1 ? kV : (g + 1) * p.cg - q.c;
#pragma unroll
    for (int i = 0; i < kV; ++i) {
        if (left == 0) { ++g; left = p.cg; }
        fn(i, g);
        --left;
    }
}

constexpr int kGnRows = 8;           // rows of a chunk

// A slice's statistics: of each group of a bundle (or the part of one) the mean and the squares about it
template <typename T, int kV> __global__ __launch_bounds__(kBlock) void gn_stats_kernel(const GnArgs p) {
    __shared__ float s_mean[kBlock * kV + 2], s_square[kBlock * kV + 2];
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
    // each channel over the rows of threads
    const int len = q.end - q.begin, wide = p.group_parts > 1 ? q.width : p.cg, least = len / q.rows, longer = len % q.rows;
    const float len_share = 1.0f / (float)len;
    float c_mean[2], c_square[2];                                    // (a bundle has 512 channels at most)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        const int c = (int)threadIdx.x + e * kBlock;
        c_mean[e] = c_square[e] = 0.0f;
        if (c >= q.width) break;
        for (int r = 0; r < q.rows; ++r) c_mean[e] = fmaf((float)(least + (r < longer)), s_mean[r * pitch + c], c_mean[e]);
        c_mean[e] *= len_share;
        for (int r = 0; r < q.rows; ++r) {
            const float held = (float)(least + (r < longer)), off = s_mean[r * pitch + c] - c_mean[e];
            c_square[e] += fmaf(held * off, off, held > 0.0f ? s_square[r * pitch + c] : 0.0f);
        }
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        const int c = (int)threadIdx.x + e * kBlock;
        if (c >= q.width) break;
        s_mean[c] = c_mean[e];
        s_square[c] = c_square[e];
    }
    __syncthreads();
    // a team of lanes to a group of the bundle: its channels
    int lanes = kWave;
    while (lanes > 1 && lanes * q.k > kBlock) lanes /= 2;
    const int team = (int)threadIdx.x / lanes, lane = (int)threadIdx.x % lanes;
    for (int j0 = 0; j0 < q.k; j0 += kBlock / lanes) {               // (as often for every lane)
        const int j = min(j0 + team, q.k - 1);
        float sum = 0.0f;
        for (int c = lane; c < wide; c += lanes) sum += s_mean[j * wide + c];
        for (int over = 1; over < lanes; over *= 2) sum += __shfl_xor(sum, over, kWave);
        const float mean = sum / (float)wide;
        sum = 0.0f;
        for (int c = lane; c < wide; c += lanes) {
            const float off = s_mean[j * wide + c] - mean;
            sum += fmaf((float)len * off, off, s_square[j * wide + c]);
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
    const int n = p.group_parts * p.part_slices;
    const float2 *from = p.parts + unit * n;
    auto held = [&](int e) {
        int width = p.cg;
        if (p.group_parts > 1) {
            const int part = e / p.part_slices;
            e -= part * p.part_slices;
            width = min(p.width, p.cg - part * p.width);
        }
        return (float)min(p.part_slice, p.positions - e * p.part_slice) * (float)width;
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
    return make_float2(mean, __builtin_amdgcn_rsqf(sum / count + p.eps));
}

constexpr int kGnMaxGroups = 512;    // of a bundle

template <typename T, int kV> __global__ __launch_bounds__(kBlock) void gn_apply_kernel(const GnArgs p) {
    __shared__ float2 s_stats[kGnMaxGroups];
    const GnPlace q = gn_place<kV>(p);
    const int64_t at = q.n * p.positions * p.channels + q.c0 + q.c;
    const T *x = (const T *)p.x + at;
    T *out = (T *)p.out + at;
    RowPiece<T, kV> rows[kGnRows];
    auto request = [&](int t) {
#pragma unroll
        for (int k = 0; k < kGnRows; ++k) rows[k] = load_row_piece<T, kV>(x + (int64_t)min(t + k * q.rows, q.end - 1) * p.channels);
    };
    if (q.there) request(q.begin + q.row);                           // on their way while the statistics are joined
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
    float w[kV], b[kV], mean[kV];
    if (q.there) gn_weights<T, kV>(p, q.c0 + q.c, w, b);
    __syncthreads();
    if (!q.there) return;
    gn_by_group<kV>(p, q, [&](int i, int g) {
        mean[i] = s_stats[g].x;
        w[i] *= s_stats[g].y;
    });
    for (int t = q.begin + q.row; t < q.end; t += kGnRows * q.rows) {
        if (t != q.begin + q.row) request(t);
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
        gn_by_group<kV>(p, q, [&](int i, int g) {
            const int64_t unit = q.n * p.groups + q.g0 + g;
            mean[i] = p.read_stats[unit].x;
            rstd[i] = p.read_stats[unit].y;
            m1[i] = m2[i] = 0.0f;
            if constexpr (!kSums) {
                m1[i] = p.means[unit].x;
                m2[i] = p.means[unit].y;
            }
        });
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
    a.cols = (a.width + v - 1) / v;
    return true;
}

// Slices of whole chunks of a workgroup's rows, as long as there are `enough` workgroups; false: too many.  768 for the statistics, 1024 for the gradients' sums, 2048 for values and dx: maps of 56 x 56 x 192
// in fp16, half as many of each and twice as many: 32 of them 26.1 us, 27.7 and 26.1; 64 44.9, 47.6 and 52.8; with gradients 32 81.3, 79.8 and 81.4; 64 123.6, 121.8 and 137.9.
static bool gn_cut(GnArgs &a, int64_t enough) {
    const int64_t chunk = (int64_t)(kBlock / a.cols) * kGnRows, others = a.batch * a.bundles, chunks = (a.positions + chunk - 1) / chunk;
    int64_t each = chunks * others / enough;
    each = each < 1 ? 1 : each < chunks ? each : chunks;
    a.slice = (int)(each * chunk < a.positions ? each * chunk : a.positions);
    a.slices = (int)((a.positions + (int64_t)a.slice - 1) / a.slice);
    return others * a.slices <= kGnLaunch / kBlock;
}
// The statistics', and then the values' slices, whose workgroups all join the statistics' parts
static bool gn_cut_stats(GnArgs &a) {
    if (!gn_cut(a, 768)) return false;
    a.part_slices = a.slices;
    a.part_slice = a.slice;
    return true;
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
    if (!gn_slices(a, gn_size(params->dtype)) || !gn_cut_stats(a)) return SS2D_ENOTSUP;
    return a.batch * a.groups * a.group_parts * a.part_slices * 8;
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
            constexpr int kK = decltype(k)::value;
            const int64_t wanted = kGnThreads / ((int64_t)kLanes * a.groups);
            a.samples = (int)(wanted < 1 ? 1 : wanted < a.batch ? wanted : a.batch);
            const int64_t wgs = ((int64_t)a.samples * a.groups + kTeams - 1) / kTeams;
            if (wgs > kGnLaunch / kBlock) return (int)SS2D_ENOTSUP;
            gn_unit_kernel<decltype(t), decltype(vec)::value, kLanes, kK><<<(uint32_t)wgs, kBlock, 0, st>>>(a);
            return launch_status();
        });
    if (!gn_slices(a, size) || !gn_cut_stats(a)) return SS2D_ENOTSUP;
    if (!workspace || reinterpret_cast<uintptr_t>(workspace) % 16) return SS2D_EINVAL;
    if (workspace_bytes < a.batch * a.groups * a.group_parts * a.part_slices * 8) return SS2D_ENOMEM;
    a.parts = (float2 *)workspace;
    return gn_sliced(params->dtype, a.channels, [&](auto t, auto vec) {
        gn_stats_kernel<decltype(t), decltype(vec)::value><<<(uint32_t)(a.batch * a.bundles * a.slices), kBlock, 0, st>>>(a);
        if (!gn_cut(a, 2048)) return (int)SS2D_ENOTSUP;
        gn_apply_kernel<decltype(t), decltype(vec)::value><<<(uint32_t)(a.batch * a.bundles * a.slices), kBlock, 0, st>>>(a);
        return launch_status();
    });
}

static int64_t gn_bwd_plan(const ss2d_group_norm_bwd_params *params, GnArgs &a, int &lanes, int &each) {
    const ss2d_group_norm_params *p = &params->fwd;
    if ((params->dweight || params->dbias) && (a.channels + (int64_t)kWave - 1) / kWave > kGnLaunch / 1024) return SS2D_ENOTSUP;       // (more channels than gn_sum_kernel's launch counts)
    const int v = gn_vec(a.cg, gn_size(p->dtype));
    if (a.positions == 1 && gn_unit(a, v, lanes, each)) {
        a.samples = gn_samples(a, lanes);
        return (int64_t)a.samples * 2 * a.channels * 4;
    }
    lanes = 0;
    if (!gn_slices(a, gn_size(p->dtype)) || !gn_cut(a, 1024)) return SS2D_ENOTSUP;
    return (a.batch * a.slices * 2 * a.channels * 4 + 15) / 16 * 16 + a.batch * a.groups * 8;
}

extern "C" int64_t ss2d_group_norm_bwd_workspace_bytes(const ss2d_group_norm_bwd_params *params) {
    GnArgs a;
    const int rc = gn_read(params ? &params->fwd : nullptr, a);
    if (rc != SS2D_OK) return rc;
    int lanes, each;
    return a.batch == 0 || a.positions == 0 ? 0 : gn_bwd_plan(params, a, lanes, each);
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
    const int64_t need = gn_bwd_plan(params, a, lanes, each);
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
            constexpr int kK = decltype(k)::value, kUnits = kK == 1 ? 2 : 1;
            gn_unit_grad_kernel<decltype(t), decltype(vec)::value, kLanes, kK, kUnits><<<(uint32_t)wgs, kBlock, 0, st>>>(a);
            return launch_status();
        });
    } else {
        parts = a.batch * a.slices;
        a.means = (float2 *)((uint8_t *)workspace + (parts * 2 * a.channels * 4 + 15) / 16 * 16);
        const int64_t teams = (a.batch * a.groups + kBlock / kWave - 1) / (kBlock / kWave);
        if (teams > kGnLaunch / kBlock) return SS2D_ENOTSUP;
        status = gn_sliced(dtype, a.channels, [&](auto t, auto vec) {
            gn_slice_grad_kernel<decltype(t), decltype(vec)::value, true><<<(uint32_t)(a.batch * a.bundles * a.slices), kBlock, 0, st>>>(a);
            gn_means_kernel<decltype(t)><<<(uint32_t)teams, kBlock, 0, st>>>(a);
            if (!gn_cut(a, 2048)) return (int)SS2D_ENOTSUP;
            gn_slice_grad_kernel<decltype(t), decltype(vec)::value, false><<<(uint32_t)(a.batch * a.bundles * a.slices), kBlock, 0, st>>>(a);
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
