// Linear attention with a decay for each head: tables of the chunks, the walk over the states, outputs (the mathematics is in
// linear_attention.h).
#include "linear_attention.h"

namespace ss2d {

// ---- tables -------------------------------------------------------------------------------------------------------------------------
// Packed sequences: their places from cu, made ascending and held inside the rows whatever cu holds, and where their chunks and
// segments begin.  One workgroup, 256 sequences at a time.
__global__ __launch_bounds__(kBlock) void la_sequences_kernel(const LaArgs p, int chunk) {
    __shared__ int most[kBlock], n_chunks[kBlock], n_segs[kBlock];
    const int tid = threadIdx.x;
    int carry = 0, chunks = 0, segs = 0, first = 0;
    for (int base = 0; base < p.n_seqs; base += kBlock) {
        const int n = base + tid;
        const bool in = n < p.n_seqs;
        auto place = [&](int i) { const int c = p.cu[i]; return c < 0 ? 0 : c < p.tokens ? c : p.tokens; };
        most[tid] = in ? place(n) : 0;
        __syncthreads();
        for (int d = 1; d < kBlock; d *= 2) {
            const int other = tid >= d ? most[tid - d] : 0;
            __syncthreads();
            most[tid] = max(most[tid], other);
            __syncthreads();
        }
        const int start = max(carry, most[tid]), end = in ? max(start, place(n + 1)) : start;
        const int mine = (end - start + chunk - 1) / chunk, parts = in ? max(1, (mine + p.seg_chunks - 1) / p.seg_chunks) : 0;
        n_chunks[tid] = mine;
        n_segs[tid] = parts;
        __syncthreads();
        for (int d = 1; d < kBlock; d *= 2) {
            const int a = tid >= d ? n_chunks[tid - d] : 0, b = tid >= d ? n_segs[tid - d] : 0;
            __syncthreads();
            n_chunks[tid] += a;
            n_segs[tid] += b;
            __syncthreads();
        }
        if (in) p.seqs[n] = make_int4(start, end, chunks + n_chunks[tid] - mine, segs + n_segs[tid] - parts);
        chunks += n_chunks[kBlock - 1];
        segs += n_segs[kBlock - 1];
        __syncthreads();
        most[tid] = end;                                             // (of a thread without a sequence: an earlier one's start)
        if (base == 0 && tid == 0) n_chunks[0] = start;
        __syncthreads();
        if (base == 0) first = n_chunks[0];
        const int last = min(p.n_seqs - base, kBlock) - 1;
        carry = most[last];
        __syncthreads();
    }
    if (tid == 0) p.seqs[p.n_seqs] = make_int4(first, carry, chunks, segs);
}

// Chunk c's entry of the table.  Behind the sequences' chunks come those of the rows of no sequence, then none.
__device__ __forceinline__ int4 la_find_chunk(const LaArgs &p, int c, int chunk) {
    if (!p.cu) {
        const int n = c / p.per_seq, t = (c - n * p.per_seq) * chunk;
        return make_int4(n, t, min(chunk, p.tokens - t), n);
    }
    const int4 all = p.seqs[p.n_seqs];
    if (c < all.z) {
        int lo = 0, hi = p.n_seqs;                                   // the last sequence whose first chunk is not behind c
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if (p.seqs[mid].z <= c) lo = mid; else hi = mid;
        }
        const int4 s = p.seqs[lo];
        const int t = s.x + (c - s.z) * chunk;
        return make_int4(0, t, min(chunk, s.y - t), lo);
    }
    const int before = (all.x + chunk - 1) / chunk;
    int t = (c - all.z) * chunk, end = all.x;
    if (c - all.z >= before) { t = all.y + (c - all.z - before) * chunk; end = p.tokens; }
    return make_int4(0, t, max(0, min(chunk, end - t)), -1);
}

// The chunks' entries and decays: C lanes to a chunk and head, sums in 64 bits.
template <int kChunk>
__global__ __launch_bounds__(kBlock) void la_chunks_kernel(const LaArgs p, int64_t total) {
    const int t = threadIdx.x % kChunk;
    const int64_t id = (int64_t)blockIdx.x * (kBlock / kChunk) + threadIdx.x / kChunk;
    if (id >= total) return;
    const int c = (int)(id / p.heads), h = (int)(id - (int64_t)c * p.heads);
    const int4 e = la_find_chunk(p, c, kChunk);
    if (h == 0 && t == 0) p.chunks[c] = e;
    double sum = 0.0;
    if (p.decay && t < e.z && e.w >= 0) {
        const double g = (double)load_decay(p.decay, e.x * p.decay_batch + (int64_t)(e.y + t) * p.decay_token + h * p.decay_head, p.decay_dtype) * 1.4426950408889634;
        sum = g < -65536.0 ? -65536.0 : g;                           // exp of either is 0; sums stay finite
    }
#pragma unroll
    for (int d = 1; d < kChunk; d *= 2) {
        const double other = __shfl_up(sum, d, kChunk);
        if (t >= d) sum += other;
    }
    const float high = (float)sum;
    p.cum[id * kChunk + t] = make_float2(high, (float)(sum - (double)high));
}

// ---- the walk over the states ------------------------------------------------------------------------------------------------------
// A workgroup owns a 64 x 64 piece of one head's state, in accumulators (wavefront w rows 16 w .. of a's dimension), and walks a segment of
// a sequence's chunks.  kLocal: a segment's own sum alone, from zero, and its decay, so that la_join_kernel can tell every segment
// what comes in.  The next chunk's rows are on their way while this one is added.
// For 16-bit operands the weighted one is split into two bf16 values: states are good to 2^-17.
template <typename Op, typename T, bool kLocal>
__global__ __launch_bounds__(kBlock) void la_walk_kernel(const LaArgs p, const LaWalk w, uint32_t total) {
    using E = typename Op::E;
    using Frag = typename Op::Frag;
    constexpr int kC = Op::kChunk, kPitch = kLaTile + Op::kPad, kVec = kVecOf<T>, kPerRow = kLaTile / kVec, kN = kC * kPerRow / kBlock;
    constexpr bool kSplit = sizeof(E) == 2;
    __shared__ __align__(16) E at[kC * kPitch], al[kSplit ? kC * kPitch : 1], bt[kC * kPitch];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int tiles_a = (w.a.dim + kLaTile - 1) / kLaTile, tiles = tiles_a * ((w.b.dim + kLaTile - 1) / kLaTile);
    const uint32_t id = xcd_contiguous_id(blockIdx.x, total);
    const int tile = id % (uint32_t)tiles, h = id / (uint32_t)tiles % (uint32_t)p.heads, seg = id / (uint32_t)tiles / (uint32_t)p.heads;
    const int a0 = tile % tiles_a * kLaTile, b0 = tile / tiles_a * kLaTile;
    int n;
    if (p.cu) {
        if (seg >= p.seqs[p.n_seqs].w) return;
        int lo = 0, hi = p.n_seqs;
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if (p.seqs[mid].w <= seg) lo = mid; else hi = mid;
        }
        n = lo;
    } else n = seg / p.segs_per_seq;
    const int4 s = la_sequence(p, n);
    const int n_chunks = (s.y - s.x + kC - 1) / kC, begin = (seg - s.w) * p.seg_chunks, count = min(p.seg_chunks, n_chunks - begin);
    const bool lone = n_chunks <= p.seg_chunks;                      // the sequence has this one segment
    const bool last = w.reverse ? begin == 0 : begin + count >= n_chunks;
    const int64_t b = p.cu ? 0 : n;
    const T *pa = reinterpret_cast<const T *>(w.a.p) + b * w.a.batch + (int64_t)(h / w.a.div) * w.a.head + a0;
    const T *pb = reinterpret_cast<const T *>(w.b.p) + b * w.b.batch + (int64_t)(h / w.b.div) * w.b.head + b0;

    floatx4_t acc[4];                                                // element (16 wave + 4 (lane / 16) + v, 16 i + lane % 16)
    const int ia = a0 + 16 * wave + 4 * (lane >> 4), ib = b0 + (lane & 15);
    float *local = p.local + (((int64_t)seg * p.heads + h) * tiles + tile) * (kLaTile * kLaTile);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        acc[i] = floatx4_t{0, 0, 0, 0};
        if constexpr (!kLocal) {
            if (!lone) acc[i] = *reinterpret_cast<const floatx4_t *>(local + i * 4 * kBlock + 4 * tid);
            else if (w.from)
#pragma unroll
                for (int v = 0; v < 4; ++v)
                    if (ia + v < w.a.dim && ib + 16 * i < w.b.dim)
                        acc[i][v] = w.from[((int64_t)n * p.heads + h) * p.k.dim * p.v.dim + (ia + v) * w.from_a + (ib + 16 * i) * w.from_b];
        }
    }
    if (kLocal && lone) return;

    u32x4_t ra[kN], rb[kN];
    float weight[kN], decay = 1.0f;
    double sum = 0.0;
    auto fetch = [&](int i) {                                        // the i-th chunk of the walk
        const int c = begin + (w.reverse ? count - 1 - i : i), t0 = s.x + c * kC, len = min(kC, s.y - t0);
        const float2 *cum = p.cum + ((int64_t)(s.z + c) * p.heads + h) * kC;
        const float2 end = cum[kC - 1];
        if constexpr (kLocal) sum += (double)end.x + (double)end.y;
#pragma unroll
        for (int j = 0; j < kN; ++j) {
            const int at_ = tid + j * kBlock, row = at_ / kPerRow, col = at_ % kPerRow * kVec;
            ra[j] = rb[j] = u32x4_t{0, 0, 0, 0};
            if (row < len) {
                ra[j] = load_piece(pa + (int64_t)(t0 + row) * w.a.token, col, w.a.dim - a0, w.a.aligned);
                rb[j] = load_piece(pb + (int64_t)(t0 + row) * w.b.token, col, w.b.dim - b0, w.b.aligned);
            }
            const float2 g = cum[row];
            weight[j] = w.reverse ? p.scale * exp2f(g.x + g.y) : exp2f((end.x - g.x) + (end.y - g.y));
        }
        decay = exp2f(end.x + end.y);
    };
    if (count > 0) fetch(0);
    for (int i = 0; i < count; ++i) {
        const int64_t at_chunk = (int64_t)(s.z + begin + (w.reverse ? count - 1 - i : i)) * p.heads + h;
#pragma unroll
        for (int j = 0; j < kN; ++j) {
            const int at_ = tid + j * kBlock, row = at_ / kPerRow, col = at_ % kPerRow * kVec;
            put_piece<T, E>(bt + row * kPitch + col, rb[j]);
            if constexpr (kSplit) {
                u32x4_t hi, lo;
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const float x = unpack_lo<T>(ra[j][q]) * weight[j], y = unpack_hi<T>(ra[j][q]) * weight[j];
                    hi[q] = pack2_from_f32<bf16_t>(x, y);
                    const float xh = unpack_lo<bf16_t>(hi[q]), yh = unpack_hi<bf16_t>(hi[q]);
                    lo[q] = pack2_from_f32<bf16_t>(fabsf(xh) <= FLT_MAX ? x - xh : 0.0f, fabsf(yh) <= FLT_MAX ? y - yh : 0.0f);
                }
                *reinterpret_cast<u32x4_t *>(at + row * kPitch + col) = hi;
                *reinterpret_cast<u32x4_t *>(al + row * kPitch + col) = lo;
            } else {
#pragma unroll
                for (int q = 0; q < kVec; q += 4)
                    *reinterpret_cast<floatx4_t *>(at + row * kPitch + col + q) =
                        floatx4_t{piece_at<T>(ra[j], q), piece_at<T>(ra[j], q + 1), piece_at<T>(ra[j], q + 2), piece_at<T>(ra[j], q + 3)} * weight[j];
            }
        }
        const float keep = decay;
        __syncthreads();
        if (i + 1 < count) fetch(i + 1);
        if constexpr (!kLocal) {                                     // the state as the chunk finds it
            const int da = la_state_dim(w.a.dim), db = la_state_dim(w.b.dim);
            E *out = reinterpret_cast<E *>(w.out) + at_chunk * da * db, *out_t = reinterpret_cast<E *>(w.out_t) + at_chunk * da * db;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (w.out && ia < da && ib + 16 * j < db) {
                    E *o = out + (int64_t)(ib + 16 * j) * da + ia;
                    Op::put4(o, acc[j]);
                    if constexpr (kSplit)
                        if (w.low) {
                            floatx4_t rest;
#pragma unroll
                            for (int v = 0; v < 4; ++v) {
                                const float high = to_f32(from_f32<bf16_t>(acc[j][v]));
                                rest[v] = fabsf(high) <= FLT_MAX ? acc[j][v] - high : 0.0f;
                            }
                            Op::put4(o + w.low, rest);
                        }
                    if (w.out_t)
#pragma unroll
                        for (int v = 0; v < 4; ++v) out_t[(int64_t)(ia + v) * db + ib + 16 * j] = from_f32<E>(acc[j][v]);
                }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[j] *= keep;
#pragma unroll
        for (int k0 = 0; k0 < kC; k0 += Op::kStep) {
            const Frag fa = Op::cols(at, kPitch, 16 * wave, k0, lane);
            Frag fl;
            if constexpr (kSplit) fl = Op::cols(al, kPitch, 16 * wave, k0, lane);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const Frag fb = Op::cols(bt, kPitch, 16 * j, k0, lane);
                acc[j] = Op::mma(fa, fb, acc[j]);
                if constexpr (kSplit) acc[j] = Op::mma(fl, fb, acc[j]);
            }
        }
        __syncthreads();
    }
    if constexpr (kLocal) {
#pragma unroll
        for (int i = 0; i < 4; ++i) *reinterpret_cast<floatx4_t *>(local + i * 4 * kBlock + 4 * tid) = acc[i];
        if (tile == 0 && tid == 0) p.local[(int64_t)p.max_segs * p.heads * tiles * (kLaTile * kLaTile) + (int64_t)seg * p.heads + h] = exp2f((float)sum);
    } else if (w.to && last) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int v = 0; v < 4; ++v)
                if (ia + v < w.a.dim && ib + 16 * i < w.b.dim)
                    w.to[((int64_t)n * p.heads + h) * p.k.dim * p.v.dim + (ia + v) * w.from_a + (ib + 16 * i) * w.from_b] = acc[i][v];
    }
}

// What comes into each segment of a sequence, from the segments' own sums: in their place.
__global__ __launch_bounds__(kBlock) void la_join_kernel(const LaArgs p, const LaWalk w, int chunk) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int tiles_a = (w.a.dim + kLaTile - 1) / kLaTile, tiles = tiles_a * ((w.b.dim + kLaTile - 1) / kLaTile);
    const int tile = blockIdx.x % (uint32_t)tiles, h = blockIdx.x / (uint32_t)tiles % (uint32_t)p.heads, n = blockIdx.x / (uint32_t)tiles / (uint32_t)p.heads;
    const int4 s = la_sequence(p, n);
    const int n_chunks = (s.y - s.x + chunk - 1) / chunk, segs = (n_chunks + p.seg_chunks - 1) / p.seg_chunks;
    if (segs <= 1) return;
    const int ia = tile % tiles_a * kLaTile + 16 * wave + 4 * (lane >> 4), ib = tile / tiles_a * kLaTile + (lane & 15);
    const float *decays = p.local + (int64_t)p.max_segs * p.heads * tiles * (kLaTile * kLaTile);
    for (int i = 0; i < 4; ++i) {
        floatx4_t state = {0, 0, 0, 0};
        if (w.from)
            for (int v = 0; v < 4; ++v)
                if (ia + v < w.a.dim && ib + 16 * i < w.b.dim)
                    state[v] = w.from[((int64_t)n * p.heads + h) * p.k.dim * p.v.dim + (ia + v) * w.from_a + (ib + 16 * i) * w.from_b];
        for (int q = 0; q < segs; ++q) {
            const int64_t seg = s.w + (w.reverse ? segs - 1 - q : q);
            floatx4_t *at = reinterpret_cast<floatx4_t *>(p.local + ((seg * p.heads + h) * tiles + tile) * (kLaTile * kLaTile) + i * 4 * kBlock + 4 * tid);
            const floatx4_t own = *at;
            *at = state;
            state = state * decays[seg * p.heads + h] + own;
        }
    }
}

template <typename Op, typename T> int la_walk(const LaArgs &p, const LaWalk &w, void *stream) {
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    const int64_t tiles = (int64_t)((w.a.dim + kLaTile - 1) / kLaTile) * ((w.b.dim + kLaTile - 1) / kLaTile);
    const int64_t total = (int64_t)p.max_segs * p.heads * tiles;
    if (total > 0x7fffffff) return SS2D_EINVAL;
    if (p.max_segs > p.n_seqs) {
        la_walk_kernel<Op, T, true><<<(uint32_t)total, kBlock, 0, st>>>(p, w, (uint32_t)total);
        la_join_kernel<<<(uint32_t)((int64_t)p.n_seqs * p.heads * tiles), kBlock, 0, st>>>(p, w, Op::kChunk);
    }
    la_walk_kernel<Op, T, false><<<(uint32_t)total, kBlock, 0, st>>>(p, w, (uint32_t)total);
    return launch_status();
}
template int la_walk<OperandF32, float>(const LaArgs &, const LaWalk &, void *);
template int la_walk<OperandF32, f16_t>(const LaArgs &, const LaWalk &, void *);
template int la_walk<OperandBf16, bf16_t>(const LaArgs &, const LaWalk &, void *);

// ---- outputs -----------------------------------------------------------------------------------------------------------------------
// A workgroup owns a chunk of one head.  Its wavefronts take the weights of the chunk's pairs 16 tokens each, then the output's columns 16 each: the
// states are read from memory straight into operands, each value once.  Products come out transposed (lane: one token, four
// neighbouring values), so that what a token has to be multiplied with is one value of the lane and stores are 8 or 16 bytes.
// The weights behind the diagonal are zeros; a product of zero with what is infinite or NaN would reach tokens in front of it, so a
// chunk that holds such a value sums its pairs one by one.
template <typename Op, typename T>
__global__ __launch_bounds__(kBlock) void la_out_kernel(const LaArgs p, uint32_t total, FastDiv per_key, FastDiv per_value) {
    using E = typename Op::E;
    using Frag = typename Op::Frag;
    constexpr int kC = Op::kChunk, kM = kC / 16, kVec = kVecOf<T>, kPitchP = kC + Op::kPad;
    extern __shared__ __align__(16) char lds[];
    const int dk = la_up(p.k.dim, Op::kStep), dv = la_up(p.v.dim, 16), pitch_k = dk + Op::kPad, pitch_v = dv + Op::kPad;
    E *qt = reinterpret_cast<E *>(lds), *kt = qt + kC * pitch_k, *vt = kt + kC * pitch_k, *pt = vt + kC * pitch_v;
    float2 *cum = reinterpret_cast<float2 *>(pt + kC * kPitchP);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 15, quad = 4 * (lane >> 4);
    const uint32_t id = xcd_contiguous_id(blockIdx.x, total);
    const int c = id / (uint32_t)p.heads, h = id - (uint32_t)c * (uint32_t)p.heads;
    const int4 e = p.chunks[c];
    if (e.z <= 0) return;
    T *out = reinterpret_cast<T *>(p.out.p) + e.x * p.out.batch + (int64_t)e.y * p.out.token + (int64_t)h * p.out.head;
    if (e.w < 0) {                                                   // rows of no sequence
        for (int i = tid; i < e.z * p.v.dim; i += kBlock) out[i / p.v.dim * p.out.token + i % p.v.dim] = from_f32<T>(0.0f);
        return;
    }
    auto load = [&](const LaSide &side, E *tile, int pitch, const FastDiv &per_row) {
        const T *src = reinterpret_cast<const T *>(side.p) + e.x * side.batch + (int64_t)e.y * side.token + (int64_t)(h / side.div) * side.head;
        bool bad = false;
        for (uint32_t i = tid; i < kC * per_row.d; i += 4 * kBlock) {
            u32x4_t piece[4];
            uint32_t row[4], at[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                divmod(i + j * kBlock, per_row, row[j], at[j]);
                piece[j] = u32x4_t{0, 0, 0, 0};
                if ((int)row[j] < e.z) piece[j] = load_piece(src + (int64_t)row[j] * side.token, at[j] * kVec, side.dim, side.aligned);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (row[j] < kC) {
                    put_piece<T, E>(tile + row[j] * pitch + at[j] * kVec, piece[j]);
                    bad |= piece_bad<T>(piece[j]);
                }
        }
        return bad;
    };
    if (tid < kC) cum[tid] = p.cum[((int64_t)c * p.heads + h) * kC + tid];
    load(p.q, qt, pitch_k, per_key);
    load(p.k, kt, pitch_k, per_key);
    const bool bad = __syncthreads_or(load(p.v, vt, pitch_v, per_value));

    // weights of the pairs, P[t][s]
#pragma unroll
    for (int i = 0; i < kM * kM / 4; ++i) {
        const int tt = wave % kM, ts = wave / kM + i * (4 / kM);
        floatx4_t acc = {0, 0, 0, 0};
        if (ts <= tt) {
            for (int k0 = 0; k0 < dk; k0 += Op::kStep)
                acc = Op::mma(Op::rows(kt, pitch_k, 16 * ts, k0, lane), Op::rows(qt, pitch_k, 16 * tt, k0, lane), acc);
            const int t = 16 * tt + col, s = 16 * ts + quad;
            const float2 gt = cum[t];
#pragma unroll
            for (int v = 0; v < 4; ++v) {
                const float2 gs = cum[s + v];
                acc[v] = s + v <= t ? acc[v] * exp2f((gt.x - gs.x) + (gt.y - gs.y)) : 0.0f;
            }
        }
        Op::put4(pt + (16 * tt + col) * kPitchP + 16 * ts + quad, acc);
    }
    __syncthreads();

    const int4 s = la_sequence(p, e.w);
    const bool carried = e.y != s.x || p.initial;                    // a state comes in
    const int da = la_state_dim(p.k.dim), db = la_state_dim(p.v.dim);
    const E *states = reinterpret_cast<const E *>(p.states) + ((int64_t)c * p.heads + h) * da * db;
    for (int n = wave; 16 * n < dv; n += 4) {
        floatx4_t acc[kM];
#pragma unroll
        for (int m = 0; m < kM; ++m) acc[m] = floatx4_t{0, 0, 0, 0};
        if (carried) {
            for (int k0 = 0; k0 < dk; k0 += Op::kStep) {
                const Frag a = Op::rows(states, da, 16 * n, k0, lane);
#pragma unroll
                for (int m = 0; m < kM; ++m) acc[m] = Op::mma(a, Op::rows(qt, pitch_k, 16 * m, k0, lane), acc[m]);
            }
#pragma unroll
            for (int m = 0; m < kM; ++m) {
                const float2 g = cum[16 * m + col];
                acc[m] *= exp2f(g.x + g.y);
            }
        }
        if (!bad) {
#pragma unroll
            for (int k0 = 0; k0 < kC; k0 += Op::kStep) {
                const Frag a = Op::cols(vt, pitch_v, 16 * n, k0, lane);
#pragma unroll
                for (int m = k0 / 16; m < kM; ++m) acc[m] = Op::mma(a, Op::rows(pt, kPitchP, 16 * m, k0, lane), acc[m]);
            }
        } else {
#pragma unroll
            for (int m = 0; m < kM; ++m)
                for (int r = 0; r <= 16 * m + col; ++r) {
                    const float weight = to_f32(pt[(16 * m + col) * kPitchP + r]);
#pragma unroll
                    for (int v = 0; v < 4; ++v) acc[m][v] += weight * to_f32(vt[r * pitch_v + 16 * n + quad + v]);
                }
        }
#pragma unroll
        for (int m = 0; m < kM; ++m) {
            const int t = 16 * m + col;
            if (t < e.z) store4(out + (int64_t)t * p.out.token + 16 * n + quad, acc[m] * p.scale, p.v.dim - 16 * n - quad, p.out.aligned);
        }
    }
}

// ---- host ----------------------------------------------------------------------------------------------------------------------------
// Segments: where the sequences alone do not give the chip its workgroups, each is cut so that they do, into eight chunks at least:
// a segment is walked twice.
int la_plan(LaArgs &p, int chunk) {
    const int64_t tiles = (int64_t)((p.k.dim + kLaTile - 1) / kLaTile) * ((p.v.dim + kLaTile - 1) / kLaTile);
    const int64_t alone = (int64_t)p.n_seqs * p.heads * tiles, want = alone >= 512 ? 1 : (1024 + p.heads * tiles - 1) / (p.heads * tiles);
    const int64_t per_seq = ((int64_t)p.tokens + chunk - 1) / chunk;
    int64_t chunks, segs, seg_chunks;
    if (p.cu) {
        chunks = (int64_t)p.tokens / chunk + p.n_seqs + 2;
        seg_chunks = want == 1 ? per_seq : (per_seq + want - 1) / want;
        seg_chunks = seg_chunks < 8 ? 8 : seg_chunks;
        segs = per_seq <= seg_chunks ? p.n_seqs : chunks / seg_chunks + p.n_seqs;
    } else {
        chunks = per_seq * p.n_seqs;
        const int64_t each = (want + p.n_seqs - 1) / p.n_seqs;
        seg_chunks = (per_seq + each - 1) / each;
        seg_chunks = seg_chunks < 8 ? 8 : seg_chunks;
        p.segs_per_seq = per_seq <= seg_chunks ? 1 : (int)((per_seq + seg_chunks - 1) / seg_chunks);
        segs = (int64_t)p.segs_per_seq * p.n_seqs;
    }
    if (chunks * p.heads > 0x7fffffff / 4 || segs * p.heads * tiles > 0x7fffffff) return SS2D_EINVAL;
    p.per_seq = (int)per_seq;
    p.max_chunks = (int)chunks;
    p.seg_chunks = (int)seg_chunks;
    p.max_segs = (int)segs;
    return SS2D_OK;
}

int la_tables(const LaArgs &p, int chunk, void *stream) {
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    if (p.cu) la_sequences_kernel<<<1, kBlock, 0, st>>>(p, chunk);
    const int64_t total = (int64_t)p.max_chunks * p.heads;
    if (total == 0) return launch_status();
    const int64_t per = kBlock / chunk, grid = (total + per - 1) / per;
    if (chunk == 64) la_chunks_kernel<64><<<(uint32_t)grid, kBlock, 0, st>>>(p, total);
    else la_chunks_kernel<32><<<(uint32_t)grid, kBlock, 0, st>>>(p, total);
    return launch_status();
}

template <typename Op, typename T> static int la_forward(const LaArgs &p, void *stream) {
    int rc = la_tables(p, Op::kChunk, stream);
    if (rc != SS2D_OK) return rc;
    // with one chunk to a sequence the states that come in are none, or the initial ones, which the walk lays out
    LaWalk w = {};
    w.a = p.k; w.b = p.v;
    w.out = p.states;
    w.from = p.initial; w.to = p.final;
    w.from_a = p.v.dim; w.from_b = 1;
    const bool skip = !p.cu && p.per_seq <= 1 && !p.initial && !p.final;
    if (!skip && (rc = la_walk<Op, T>(p, w, stream)) != SS2D_OK) return rc;
    const uint32_t total = (uint32_t)p.max_chunks * (uint32_t)p.heads;
    if (total == 0) return SS2D_OK;
    const int dk = la_up(p.k.dim, Op::kStep), dv = la_up(p.v.dim, 16), c = Op::kChunk;
    const size_t bytes = sizeof(typename Op::E) * c * (2 * (dk + Op::kPad) + dv + Op::kPad + c + Op::kPad) + sizeof(float2) * c;
    // (up to 104 KB of LDS: this runtime asks for no attribute above 64)
    la_out_kernel<Op, T><<<total, kBlock, bytes, reinterpret_cast<hipStream_t>(stream)>>>(p, total, make_fastdiv(dk / kVecOf<T>), make_fastdiv(dv / kVecOf<T>));
    return launch_status();
}

static bool la_aligned(const void *p, int64_t a, int64_t b, int64_t c, int64_t bytes, int64_t size) {
    return ((uintptr_t)p | (uintptr_t)(a * size) | (uintptr_t)(b * size) | (uintptr_t)(c * size)) % bytes == 0;
}

LaSide la_side(const void *ptr, int64_t batch, int64_t token, int64_t head, int heads, int own_heads, int dim, int size, int bytes) {
    LaSide s = {};
    s.p = const_cast<void *>(ptr);
    s.batch = batch; s.token = token; s.head = head;
    s.div = own_heads > 0 ? heads / own_heads : 1;
    s.dim = dim;
    s.aligned = la_aligned(ptr, batch, token, head, bytes, size);
    return s;
}

// The arguments of a call, checked; *empty where there is nothing to do at all.
int la_arguments(const ss2d_linear_attention_params *p, LaArgs &a, bool &empty) {
    empty = false;
    if (!p) return SS2D_EINVAL;
    if (p->batch < 0 || p->seqlen < 0 || p->heads < 0 || p->n_seqs < 0 || p->key_dim < 1 || p->value_dim < 1) return SS2D_EINVAL;
    if (p->dtype < SS2D_F32 || p->dtype > SS2D_F16) return SS2D_EINVAL;
    if (p->decay && p->decay_dtype != SS2D_F32 && p->decay_dtype != p->dtype) return SS2D_EINVAL;
    if (p->q_heads < 1 || p->k_heads < 1 || p->v_heads < 1) return SS2D_EINVAL;
    if (p->heads % p->q_heads || p->heads % p->k_heads || p->heads % p->v_heads) return SS2D_EINVAL;
    if (p->cu_seqlens && (p->batch != 1 || p->n_seqs < 1)) return SS2D_EINVAL;
    if (p->key_dim > kLaMaxDim || p->value_dim > kLaMaxDim) return SS2D_ENOTSUP;
    a = {};
    a.batch = p->batch; a.tokens = p->seqlen; a.heads = p->heads;
    a.n_seqs = p->cu_seqlens ? p->n_seqs : p->batch;
    a.scale = p->scale;
    a.decay = p->decay; a.decay_dtype = p->decay_dtype;
    a.decay_batch = p->decay_batch_stride; a.decay_token = p->decay_token_stride; a.decay_head = p->decay_head_stride;
    a.cu = p->cu_seqlens;
    a.initial = p->initial_state; a.final = p->final_state;
    const int size = p->dtype == SS2D_F32 ? 4 : 2;
    a.q = la_side(p->q, p->q_batch_stride, p->q_token_stride, p->q_head_stride, p->heads, p->q_heads, p->key_dim, size, 16);
    a.k = la_side(p->k, p->k_batch_stride, p->k_token_stride, p->k_head_stride, p->heads, p->k_heads, p->key_dim, size, 16);
    a.v = la_side(p->v, p->v_batch_stride, p->v_token_stride, p->v_head_stride, p->heads, p->v_heads, p->value_dim, size, 16);
    const int64_t row = (int64_t)p->heads * p->value_dim;
    a.out = la_side(p->out, row * p->seqlen, row, p->value_dim, p->heads, p->heads, p->value_dim, size, 4 * size);
    if (a.heads == 0 || a.n_seqs == 0) { empty = true; return SS2D_OK; }
    const bool rows = a.tokens > 0;
    if (rows && (!p->q || !p->k || !p->v)) return SS2D_EINVAL;
    return la_plan(a, p->dtype == SS2D_BF16 ? OperandBf16::kChunk : OperandF32::kChunk);
}

static int64_t la_round(int64_t n) { return (n + 255) / 256 * 256; }

// Lays a call's workspace out from `base` on and says how long it is.  layouts: of states at all, of E across too; halves: 2 where what the rounding
// of states leaves is kept.
int64_t la_carve(LaArgs &p, int dtype, char *base, bool backward, bool low) {
    const int chunk = dtype == SS2D_BF16 ? OperandBf16::kChunk : OperandF32::kChunk, size = dtype == SS2D_BF16 ? 2 : 4;
    const int64_t entries = (int64_t)p.max_chunks * p.heads, state = (int64_t)la_state_dim(p.k.dim) * la_state_dim(p.v.dim);
    const int64_t tiles = (int64_t)((p.k.dim + kLaTile - 1) / kLaTile) * ((p.v.dim + kLaTile - 1) / kLaTile);
    int64_t at = 0;
    auto take = [&](auto *&ptr, int64_t bytes) {
        ptr = reinterpret_cast<std::remove_reference_t<decltype(ptr)>>(base + at);
        at += la_round(bytes);
    };
    take(p.chunks, sizeof(int4) * (int64_t)p.max_chunks);
    take(p.seqs, p.cu ? sizeof(int4) * ((int64_t)p.n_seqs + 1) : 0);
    take(p.cum, sizeof(float2) * entries * chunk);
    p.low = low ? entries * state : 0;
    take(p.states, (low ? 2 : 1) * size * entries * state);
    if (backward) {
        take(p.dstates, (low ? 2 : 1) * size * entries * state);
        take(p.dstates_t, size * entries * state);
    }
    take(p.local, p.max_segs > p.n_seqs ? 4 * (int64_t)p.max_segs * p.heads * (tiles * kLaTile * kLaTile + 1) : 0);
    return at < 256 ? 256 : at;                                      // (a caller has an address to give)
}

}  // namespace ss2d

using namespace ss2d;

extern "C" int64_t ss2d_linear_attention_workspace_bytes(const ss2d_linear_attention_params *params) {
    LaArgs a;
    bool empty;
    const int rc = la_arguments(params, a, empty);
    if (rc != SS2D_OK || empty) return rc;
    return la_carve(a, params->dtype, nullptr, false, false);
}

extern "C" int ss2d_linear_attention_fwd(const ss2d_linear_attention_params *params, void *workspace, int64_t workspace_bytes, void *stream) {
    LaArgs a;
    bool empty;
    const int rc = la_arguments(params, a, empty);
    if (rc != SS2D_OK || empty) return rc;
    if (a.tokens > 0 && !params->out) return SS2D_EINVAL;
    if (!workspace || (uintptr_t)workspace % 16 != 0) return SS2D_EINVAL;
    if (workspace_bytes < la_carve(a, params->dtype, reinterpret_cast<char *>(workspace), false, false)) return SS2D_ENOMEM;
    switch (params->dtype) {
    case SS2D_F32: return la_forward<OperandF32, float>(a, stream);
    case SS2D_F16: return la_forward<OperandF32, f16_t>(a, stream);
    default: return la_forward<OperandBf16, bf16_t>(a, stream);
    }
}
