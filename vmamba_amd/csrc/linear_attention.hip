// Linear attention with a decay for each head: tables of the chunks, the walk over the states, outputs (the mathematics is in
// linear_attention.h).
#include <type_traits>

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

// The logarithm of a token's decay
__device__ __forceinline__ float la_decay(const LaArgs &p, int64_t batch, int64_t token, int h) {
    return load_decay(p.decay, batch * p.decay_batch + token * p.decay_token + h * p.decay_head, p.decay_dtype);
}
// Their sums up to and with each of a chunk's tokens, one to a lane: in log2 units, in 64 bits, as a pair of floats.  exp2 of less than -65536 is 0 as it is of
// that, and sums stay finite.
template <int kChunk> __device__ __forceinline__ float2 la_sum_decays(float decay, int t) {
    const double g = (double)decay * 1.4426950408889634;
    double sum = g < -65536.0 ? -65536.0 : g;
#pragma unroll
    for (int d = 1; d < kChunk; d *= 2) {
        const double other = __shfl_up(sum, d, kChunk);
        if (t >= d) sum += other;
    }
    const float high = (float)sum;
    return make_float2(high, (float)(sum - (double)high));
}

// The chunks' entries and decays: C lanes to a chunk and head.  A latency: 5 us for 8192 chunks and heads.  kOut: bytes of an output's value, whose rows of no
// sequence are cleared here; 0: they are not this call's.
template <int kChunk, int kOut>
__global__ __launch_bounds__(kBlock) void la_chunks_kernel(const LaArgs p, int64_t total) {
    const int t = threadIdx.x % kChunk;
    const int64_t id = (int64_t)blockIdx.x * (kBlock / kChunk) + threadIdx.x / kChunk;
    if (id >= total) return;
    const int c = (int)(id / p.heads), h = (int)(id - (int64_t)c * p.heads);
    const int4 e = la_find_chunk(p, c, kChunk);
    if (h == 0 && t == 0) p.chunks[c] = e;
    const float2 sum = la_sum_decays<kChunk>(p.decay && t < e.z && e.w >= 0 ? la_decay(p, e.x, e.y + t, h) : 0.0f, t);
    p.cum[id * kChunk + t] = sum;
    if (t == kChunk - 1) p.kept[id] = la_kept(sum);
    if constexpr (kOut > 0) {
        using Bits = std::conditional_t<kOut == 2, uint16_t, uint32_t>;
        if (e.w >= 0) return;
        Bits *out = reinterpret_cast<Bits *>(p.out.p) + (int64_t)e.y * p.out.token + (int64_t)h * p.out.head;
        for (int r = 0; r < e.z; ++r, out += p.out.token)
            for (int d = t; d < p.v.dim; d += kChunk) out[d] = 0;
    }
}

// ---- the walk over the states ------------------------------------------------------------------------------------------------------
// Which piece of which head, and which segment of which sequence, a workgroup walks.
struct LaPlace {
    int n, h, seg, tile;
    int4 s;                          // the sequence
    int begin, count, chunks;        // of the segment, in chunks; of the sequence
};
__device__ __forceinline__ bool la_place(const LaArgs &p, uint32_t id, int tiles, int chunk, LaPlace &at) {
    at.tile = id % (uint32_t)tiles;
    at.h = id / (uint32_t)tiles % (uint32_t)p.heads;
    at.seg = id / (uint32_t)tiles / (uint32_t)p.heads;
    if (p.cu) {
        if (at.seg >= p.seqs[p.n_seqs].w) return false;
        int lo = 0, hi = p.n_seqs;
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if (p.seqs[mid].w <= at.seg) lo = mid; else hi = mid;
        }
        at.n = lo;
    } else at.n = at.seg / p.segs_per_seq;
    at.s = la_sequence(p, at.n);
    at.chunks = (at.s.y - at.s.x + chunk - 1) / chunk;
    at.begin = (at.seg - at.s.w) * p.seg_chunks;
    at.count = min(p.seg_chunks, at.chunks - at.begin);
    return true;
}

// Element (ia, ib) of the state of sequence n and head h that the caller gives or gets
__device__ __forceinline__ int64_t la_state_at(const LaArgs &p, const LaWalk &w, int n, int h, int ia, int ib) {
    return ((int64_t)n * p.heads + h) * p.k.dim * p.v.dim + ia * w.from_a + ib * w.from_b;
}

// A workgroup owns a 64 x 64 piece of one head's state, in accumulators (wavefront w rows 16 w .. of a's dimension), and walks a segment of
// a sequence's chunks.  kLocal: a segment's own sum alone, from zero, and its decay, so that la_join_kernel can tell every segment
// what comes in.  The next two chunks' rows are on their way while this one is added.  Where 16-bit states are wanted in both orders (kBoth) the products are
// made twice, with their operands exchanged: an accumulator then is four neighbours of either.  Two walks may share a launch.
// Bound by memory and by the chain of a segment's chunks, 2.6 us each.  Both walks for the gradients of 4 x 2048 tokens, 16 heads of 128 x 128, bf16: 84 us for
// 268 MB (S and E written, q, k, v and the gradient read from memory once, by the other pieces from L2), 3.2 TB/s; with E stored in both orders 102.
// A segment's own sums, 65 536 tokens, 8 heads of 64: 31 us.
template <typename Op, typename T, bool kLocal, int kParts, bool kFast, bool kBoth>
__global__ __launch_bounds__(kBlock, 2) void la_walk_kernel(const LaArgs p, const LaWalk w0, const LaWalk w1, uint32_t total) {
    using E = typename Op::E;
    using Frag = typename Op::Frag;
    constexpr int kC = Op::kChunk, kPitch = kLaTile + Op::kPad, kVec = kVecOf<T>, kPerRow = kLaTile / kVec, kN = kC * kPerRow / kBlock;
    constexpr int kTile = kLaTile * kPitch;
    constexpr bool kStaged = !kLocal && sizeof(E) == 2;              // (four floats of a lane are 16 bytes as they are)
    __shared__ __align__(16) E at[kC * kPitch], bt[kC * kPitch], st[kStaged ? (kBoth ? 4 : 2) * kTile : 1];
    __shared__ __align__(16) float weights[kC];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const bool second = blockIdx.x >= total;
    const LaWalk w = second ? w1 : w0;
    const int tiles_a = (w.a.dim + kLaTile - 1) / kLaTile, tiles = tiles_a * ((w.b.dim + kLaTile - 1) / kLaTile);
    LaPlace here;
    if (!la_place(p, xcd_contiguous_id(second ? blockIdx.x - total : blockIdx.x, total), tiles, kC, here)) return;
    const int a0 = here.tile % tiles_a * kLaTile, b0 = here.tile / tiles_a * kLaTile, h = here.h, n = here.n;
    const int4 s = here.s;
    const bool lone = here.chunks <= p.seg_chunks;                   // the sequence has this one segment
    const bool whole = w.a.dim - a0 >= kLaTile && w.b.dim - b0 >= kLaTile;           // the tiles' columns are all there
    const bool last = w.reverse ? here.begin == 0 : here.begin + here.count >= here.chunks;
    if (kLocal && (lone || last)) return;                            // (nobody asks for the last one's sum)
    const int64_t b = p.cu ? 0 : n;
    const T *pa = reinterpret_cast<const T *>(w.a.p) + b * w.a.batch + (int64_t)(h / w.a.div) * w.a.head;
    const T *pb = reinterpret_cast<const T *>(w.b.p) + b * w.b.batch + (int64_t)(h / w.b.div) * w.b.head;

    floatx4_t acc[4], turned[kBoth ? 4 : 1];                         // element (16 wave + 4 (lane / 16) + v, 16 i + lane % 16); (16 wave + lane % 16, 16 i + 4 (lane / 16) + v)
    const int quad = 4 * (lane >> 4), col = lane & 15, ia = a0 + 16 * wave + quad, ib = b0 + col, ja = a0 + 16 * wave + col, jb = b0 + quad;
    float *local = w.local + (((int64_t)here.seg * p.heads + h) * tiles + here.tile) * (kLaTile * kLaTile);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        acc[i] = floatx4_t{0, 0, 0, 0};
        if constexpr (kBoth) turned[i] = floatx4_t{0, 0, 0, 0};
        if constexpr (!kLocal) {
            if (!lone) {
                acc[i] = *reinterpret_cast<const floatx4_t *>(local + i * 4 * kBlock + 4 * tid);
                if constexpr (kBoth)
#pragma unroll
                    for (int v = 0; v < 4; ++v) turned[i][v] = local[i * 4 * kBlock + 4 * (wave * kWave + 16 * (col >> 2) + quad + v) + (col & 3)];
            } else if (w.from)
#pragma unroll
                for (int v = 0; v < 4; ++v) {
                    if (ia + v < w.a.dim && ib + 16 * i < w.b.dim) acc[i][v] = w.from[la_state_at(p, w, n, h, ia + v, ib + 16 * i)];
                    if constexpr (kBoth)
                        if (ja < w.a.dim && jb + 16 * i + v < w.b.dim) turned[i][v] = w.from[la_state_at(p, w, n, h, ja, jb + 16 * i + v)];
                }
        }
    }

    struct Rows {
        u32x4_t a[kN], b[kN];
        float weight;
        LaKeep<E> keep;
    } ring[2];
    double sum = 0.0;
    auto fetch = [&](int i, Rows &r) {                               // the i-th chunk of the walk
        const int c = here.begin + (w.reverse ? here.count - 1 - i : i), t0 = s.x + c * kC, len = min(kC, s.y - t0);
        const float2 *cum = p.cum + ((int64_t)(s.z + c) * p.heads + h) * kC;
        const float2 end = cum[kC - 1];
        if constexpr (kLocal) sum += (double)end.x + (double)end.y;
#pragma unroll
        for (int j = 0; j < kN; ++j) {
            const int at_ = tid + j * kBlock, row = at_ / kPerRow, c0 = at_ % kPerRow * kVec;
            r.a[j] = load_piece<kFast>(pa + (int64_t)t0 * w.a.token, w.a.token, row, len, a0 + c0, w.a.dim);
            r.b[j] = load_piece<kFast>(pb + (int64_t)t0 * w.b.token, w.b.token, row, len, b0 + c0, w.b.dim);
        }
        if (tid < kC) {
            const float2 g = cum[tid];
            r.weight = w.reverse ? p.scale * fast_exp2(g.x + g.y) : fast_exp2((end.x - g.x) + (end.y - g.y));
        }
        r.keep.set(end, p.kept + (int64_t)(s.z + c) * p.heads + h);
    };
    auto stage = [&](int i) {                                        // the piece before chunk i, for the stores of that chunk's step
        if constexpr (kStaged) {
            E *to = st + (i & 1) * kTile;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                Op::put4(to + (16 * j + col) * kPitch + 16 * wave + quad, acc[j]);
                if constexpr (kBoth) Op::put4(to + 2 * kTile + (16 * wave + col) * kPitch + 16 * j + quad, turned[j]);
            }
        }
    };
    auto step = [&](int i, Rows &r) {
        const int c = here.begin + (w.reverse ? here.count - 1 - i : i), len = min(kC, s.y - s.x - c * kC);
        const int64_t at_chunk = (int64_t)(s.z + c) * p.heads + h;
        if (len < kC || !whole)
#pragma unroll
            for (int j = 0; j < kN; ++j) {
                const int at_ = tid + j * kBlock, row = at_ / kPerRow, c0 = at_ % kPerRow * kVec;
                r.a[j] = held_piece<kFast, T>(r.a[j], row < len, a0 + c0, w.a.dim);
                r.b[j] = held_piece<kFast, T>(r.b[j], row < len, b0 + c0, w.b.dim);
            }
#pragma unroll
        for (int j = 0; j < kN; ++j) {
            const int at_ = tid + j * kBlock, row = at_ / kPerRow, c0 = at_ % kPerRow * kVec;
            put_piece<T, E>(at + row * kPitch + c0, r.a[j]);
            put_piece<T, E>(bt + row * kPitch + c0, r.b[j]);
        }
        if (tid < kC) weights[Op::place(tid)] = r.weight;
        const LaKeep<E> keep = r.keep;
        __syncthreads();
        if (i + 2 < here.count) fetch(i + 2, r);
        if constexpr (!kLocal) {                                     // the state as the chunk finds it, whole rows of the piece at a time
            const int da = la_state_dim(w.a.dim), db = la_state_dim(w.b.dim);
            const int64_t base = at_chunk * da * db;
            if constexpr (kStaged) {
                constexpr int kPieces = 16 / (int)sizeof(E), kRow = kLaTile / kPieces;
                const E *from = st + (i & 1) * kTile;
#pragma unroll
                for (int j = 0; j < kLaTile * kRow / kBlock; ++j) {
                    const int at_ = tid + j * kBlock, row = at_ / kRow, c0 = at_ % kRow * kPieces;
                    if (b0 + row < db && a0 + c0 < da)
                        *reinterpret_cast<u32x4_t *>(reinterpret_cast<E *>(w.out) + base + (int64_t)(b0 + row) * da + a0 + c0) = *reinterpret_cast<const u32x4_t *>(from + row * kPitch + c0);
                    if constexpr (kBoth)
                        if (w.out_t && a0 + row < da && b0 + c0 < db)
                            *reinterpret_cast<u32x4_t *>(reinterpret_cast<E *>(w.out_t) + base + (int64_t)(a0 + row) * db + b0 + c0) =
                                *reinterpret_cast<const u32x4_t *>(from + 2 * kTile + row * kPitch + c0);
                }
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (ia < da && ib + 16 * j < db) {
                        Op::put4(reinterpret_cast<E *>(w.out) + base + (int64_t)(ib + 16 * j) * da + ia, acc[j]);
                        if (w.out_t)                                 // (16 lanes are 64 bytes of a row as they are)
#pragma unroll
                            for (int v = 0; v < 4; ++v) reinterpret_cast<E *>(w.out_t)[base + (int64_t)(ia + v) * db + ib + 16 * j] = from_f32<E>(acc[j][v]);
                    }
            }
            if (sizeof(E) == 2 && w.low && ia < da)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (ib + 16 * j < db) {
                        floatx4_t rest;
#pragma unroll
                        for (int v = 0; v < 4; ++v) rest[v] = acc[j][v] - to_f32(from_f32<bf16_t>(acc[j][v]));
                        E *to = reinterpret_cast<E *>(w.out) + base + (int64_t)(ib + 16 * j) * da + ia + w.low;
                        Op::put4(to, rest);
#pragma unroll
                        for (int v = 0; v < 4; ++v) rest[v] -= to_f32(from_f32<bf16_t>(rest[v]));
                        Op::put4(to + w.low, rest);
                    }
        }
        // (in single precision a chunk's sum is made for itself: added product by product to the state, the sum of all chunks, each of them would be rounded to that)
        constexpr bool kApart = sizeof(E) == 4;
        floatx4_t mine[kApart ? 4 : 1];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if constexpr (kApart) mine[j] = floatx4_t{0, 0, 0, 0};
            else keep.scale(acc[j]);
            if constexpr (kBoth) keep.scale(turned[j]);
        }
#pragma unroll
        for (int k0 = 0; k0 < kC; k0 += Op::kStep) {
            Frag fa[kParts], fb[4];
            Op::template weigh<kParts>(Op::cols(at, kPitch, 16 * wave, k0, lane), weights + k0, lane, fa);
#pragma unroll
            for (int j = 0; j < 4; ++j) fb[j] = Op::cols(bt, kPitch, 16 * j, k0, lane);
#pragma unroll
            for (int q = 0; q < kParts; ++q)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (!kBoth && j >= 2 && w.b.dim - b0 <= 32) break;       // (nothing there)
                    floatx4_t &sum = kApart ? mine[kApart ? j : 0] : acc[j];
                    sum = Op::mma(fa[q], fb[j], sum);
                    if constexpr (kBoth) turned[j] = Op::mma(fb[j], fa[q], turned[j]);
                }
        }
        if constexpr (kApart)
#pragma unroll
            for (int j = 0; j < 4; ++j) keep.add(acc[j], mine[j]);
        stage(i + 1);
        __syncthreads();
    };
    if (here.count > 0) fetch(0, ring[0]);
    if (here.count > 1) fetch(1, ring[1]);
    stage(0);
    for (int i = 0; i < here.count; i += 2) {
        step(i, ring[0]);
        if (i + 1 < here.count) step(i + 1, ring[1]);
    }
    if constexpr (kLocal) {
#pragma unroll
        for (int i = 0; i < 4; ++i) *reinterpret_cast<floatx4_t *>(local + i * 4 * kBlock + 4 * tid) = acc[i];
        if (here.tile == 0 && tid == 0)
            w.local[(int64_t)p.max_segs * p.heads * tiles * (kLaTile * kLaTile) + (int64_t)here.seg * p.heads + h] = (float)exp2(sum);
    } else if (w.to && last) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int v = 0; v < 4; ++v)
                if (ia + v < w.a.dim && ib + 16 * i < w.b.dim) w.to[la_state_at(p, w, n, h, ia + v, ib + 16 * i)] = acc[i][v];
    }
}

// What comes into each segment of a sequence, from the segments' own sums: in their place.  A workgroup takes 16 columns of a piece; the sums of
// eight segments are on their way while eight are added (sixteen and none: 19 us instead of 16 for the 50 segments of 24 heads of 128 x 64 in the packed
// case of 12 011 tokens, 79 MB; sixteen and sixteen: 24, too few wavefronts).
constexpr uint32_t kLaJoins = 1 << 20;
__device__ __forceinline__ void la_join(const LaArgs &p, const LaWalk &w0, const LaWalk &w1, int chunk, uint32_t total, uint32_t at_block) {
    constexpr int kAhead = 8;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const bool second = at_block >= total;
    const LaWalk w = second ? w1 : w0;
    const int tiles_a = (w.a.dim + kLaTile - 1) / kLaTile, tiles = tiles_a * ((w.b.dim + kLaTile - 1) / kLaTile);
    const uint32_t block = second ? at_block - total : at_block, id = block / 4;
    const int i = block % 4, tile = id % (uint32_t)tiles, h = id / (uint32_t)tiles % (uint32_t)p.heads, n = id / (uint32_t)tiles / (uint32_t)p.heads;
    const int4 s = la_sequence(p, n);
    const int n_chunks = (s.y - s.x + chunk - 1) / chunk, segs = (n_chunks + p.seg_chunks - 1) / p.seg_chunks;
    if (segs <= 1) return;
    const int ia = tile % tiles_a * kLaTile + 16 * wave + 4 * (lane >> 4), ib = tile / tiles_a * kLaTile + 16 * i + (lane & 15);
    const float *decays = w.local + (int64_t)p.max_segs * p.heads * tiles * (kLaTile * kLaTile);
    floatx4_t state = {0, 0, 0, 0};
    if (w.from)
#pragma unroll
        for (int v = 0; v < 4; ++v)
            if (ia + v < w.a.dim && ib < w.b.dim) state[v] = w.from[la_state_at(p, w, n, h, ia + v, ib)];
    auto place = [&](int q) { return ((int64_t)s.w + (w.reverse ? segs - 1 - q : q)) * p.heads + h; };
    auto at = [&](int q) { return reinterpret_cast<floatx4_t *>(w.local + (place(q) * tiles + tile) * (kLaTile * kLaTile) + i * 4 * kBlock + 4 * tid); };
    struct Part {
        floatx4_t own[kAhead];
        float decay[kAhead];
    } ring[2];
    auto fetch = [&](int q0, Part &part) {
        if (q0 >= segs - 1) return;                                  // (the last one's sum is none)
#pragma unroll
        for (int q = 0; q < kAhead; ++q) {
            const int safe = min(q0 + q, segs - 2);
            part.own[q] = *at(safe);
            part.decay[q] = decays[place(safe)];
        }
    };
    auto step = [&](int q0, Part &part) {
#pragma unroll
        for (int q = 0; q < kAhead; ++q)
            if (q0 + q < segs) {
                *at(q0 + q) = state;
                state = state * part.decay[q] + part.own[q];
            }
    };
    fetch(0, ring[0]);
    for (int q0 = 0; q0 < segs; q0 += 2 * kAhead) {
        fetch(q0 + kAhead, ring[1]);
        step(q0, ring[0]);
        fetch(q0 + 2 * kAhead, ring[0]);
        step(q0 + kAhead, ring[1]);
    }
}
__global__ __launch_bounds__(kBlock) void la_join_kernel(const LaArgs p, const LaWalk w0, const LaWalk w1, int chunk, uint32_t total, uint32_t all) {
    for (uint32_t block = blockIdx.x; block < all; block += gridDim.x) la_join(p, w0, w1, chunk, total, block);
}

static int64_t la_tiles(const LaArgs &p) { return (int64_t)((p.k.dim + kLaTile - 1) / kLaTile) * ((p.v.dim + kLaTile - 1) / kLaTile); }

template <typename Op, typename T, bool kLocal, bool kBoth> static void la_walk_launch(const LaArgs &p, const LaWalk *w, int n, hipStream_t st) {
    constexpr int kMost = Op::kMostParts, kLess = kMost < 2 ? kMost : 2;
    const LaWalk &w0 = w[0], &w1 = w[n - 1];
    const bool fast = w0.a.pieces && w0.b.pieces && w1.a.pieces && w1.b.pieces;
    const uint32_t total = (uint32_t)((int64_t)p.max_segs * p.heads * la_tiles(p)), grid = total * (uint32_t)n;
    if (w0.exact || w1.exact) {
        if (fast) la_walk_kernel<Op, T, kLocal, kMost, true, kBoth><<<grid, kBlock, 0, st>>>(p, w0, w1, total);
        else la_walk_kernel<Op, T, kLocal, kMost, false, kBoth><<<grid, kBlock, 0, st>>>(p, w0, w1, total);
    } else {
        if (fast) la_walk_kernel<Op, T, kLocal, kLess, true, kBoth><<<grid, kBlock, 0, st>>>(p, w0, w1, total);
        else la_walk_kernel<Op, T, kLocal, kLess, false, kBoth><<<grid, kBlock, 0, st>>>(p, w0, w1, total);
    }
}

// What comes into the segments
template <typename Op, typename T> static int la_segments(const LaArgs &p, const LaWalk *w, int n, hipStream_t st) {
    if (p.max_segs <= p.n_seqs) return SS2D_OK;
    la_walk_launch<Op, T, true, false>(p, w, n, st);
    const uint32_t total = (uint32_t)((int64_t)p.n_seqs * p.heads * la_tiles(p) * 4), grid = total * (uint32_t)n;
    la_join_kernel<<<grid < kLaJoins ? grid : kLaJoins, kBlock, 0, st>>>(p, w[0], w[n - 1], Op::kChunk, total, grid);
    return launch_status();
}

template <typename Op, typename T> int la_walks(const LaArgs &p, const LaWalk *w, int n, void *stream) {
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    const int rc = la_segments<Op, T>(p, w, n, st);
    if (rc != SS2D_OK) return rc;
    constexpr bool kTurn = sizeof(typename Op::E) == 2;
    if (kTurn && (w[0].out_t || w[n - 1].out_t)) la_walk_launch<Op, T, false, kTurn>(p, w, n, st);
    else la_walk_launch<Op, T, false, false>(p, w, n, st);
    return launch_status();
}
template int la_walks<OperandF32, float>(const LaArgs &, const LaWalk *, int, void *);
template int la_walks<OperandF32, f16_t>(const LaArgs &, const LaWalk *, int, void *);
template int la_walks<OperandBf16, bf16_t>(const LaArgs &, const LaWalk *, int, void *);

// ---- outputs -----------------------------------------------------------------------------------------------------------------------
// A workgroup owns 64 values' columns of one head and walks a segment of chunks with their states, so that nothing but q, k, v and the outputs passes
// through memory.  Its eight wavefronts are two to 16 columns: of a chunk's outputs each makes half of the tokens', of the state (in
// accumulators, 32 bits) half of the keys', and the state as an operand goes from one to the other through LDS.  Per chunk: weights of its pairs,
// 16 x 16 tokens to a wavefront at a time, through LDS; out = state and pairs; then the state with the chunk's keys and weighted values.  Products come
// out transposed (lane: one token, four neighbouring values), so that what a token has to be multiplied with is one value of the lane.
// The weights behind the diagonal are zeros; a product of zero with what is infinite or NaN would reach tokens in front of it, so a
// chunk that holds such a value sums its pairs one by one.
// 8 x 4096 tokens, 16 heads of 128 x 128, bf16: 198-220 us for 555 MB, 2.7 TB/s.  Neither memory nor the matrix cores bound it (busy 12 %) but a chunk's chain -- rows to
// LDS, pairs, outputs, state, three barriers between them, 357 vector instructions of a wavefront and 2900 cycles of LDS reads -- which nothing else hides: these are
// 256 workgroups, one to a CU.  Two would fit, and 16 x 2048 tokens, which are two, take 158 us for the same work.  The call took 320 us
// with four wavefronts of all keys in place of eight of half of them, 474 with the states of all chunks through memory.
constexpr int kLaWaves = kLaThreads / kWave;
// kOwn, of sequences of a few chunks and up to 64 keys: it sums their decays itself, which takes a chunk less than another launch takes for all of them
// (37 tokens, 8 heads of 64, bf16: 10.9 -> 8.6 us a call; 120 tokens 12.2 -> 9.9, 256, four chunks, 16.6 -> 15.4).  Keys of 128 and 256 would gain as much at one or two
// chunks (11.0 -> 8.5 and 13.6 -> 10.1 at 37 tokens); the kernels of these sizes are not there twice.
constexpr int kLaOwnChunks = 4, kLaOwnKeys = 64;

template <typename Op, typename T, int kTiles, int kParts, bool kFast, bool kOwn>
__global__ __launch_bounds__(kLaThreads, kTiles <= 8 ? 4 : 2) void la_out_kernel(const LaArgs p, const LaWalk w, uint32_t total) {
    using E = typename Op::E;
    using Frag = typename Op::Frag;
    constexpr int kC = Op::kChunk, kM = kC / 16, kVec = kVecOf<T>, kKeys = 16 * kTiles, kPitchK = kKeys + Op::kPad, kPitchV = kLaTile + Op::kPad, kPitchP = kC + Op::kPad;
    constexpr int kPerKey = kKeys / kVec, kPerValue = kLaTile / kVec, kNk = (kC * kPerKey + kLaThreads - 1) / kLaThreads, kNv = (kC * kPerValue + kLaThreads - 1) / kLaThreads;
    constexpr int kHalfM = kM / 2, kHalf = kTiles / 2, kSteps = kC / Op::kStep, kPairTiles = kM * (kM + 1) / 2;
    extern __shared__ __align__(16) char lds[];
    E *qt = reinterpret_cast<E *>(lds), *kt = qt + kC * kPitchK, *st = kt + kC * kPitchK, *vt = st + kLaTile * kPitchK, *pt = vt + kC * kPitchV;
    float *weights = reinterpret_cast<float *>(pt + kC * kPitchP);   // of a token's value in the state behind the chunk
    float2 *cum = reinterpret_cast<float2 *>(weights + kC);
    int *bad = reinterpret_cast<int *>(cum + kC);
    float2 *kept = reinterpret_cast<float2 *>(bad + 2);              // (kOwn: of this chunk)
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 15, quad = 4 * (lane >> 4);
    const int mine = wave % 4, half = wave / 4;                      // columns 16 mine .., tokens and keys of this half
    const int tiles = (p.v.dim + kLaTile - 1) / kLaTile;
    LaPlace here;
    if (!la_place(p, xcd_contiguous_id(blockIdx.x, total), tiles, kC, here)) return;
    const int v0 = here.tile * kLaTile, h = here.h, n = here.n;
    const int4 s = here.s;
    const bool lone = here.chunks <= p.seg_chunks, last = here.begin + here.count >= here.chunks, live = v0 + 16 * mine < p.v.dim;
    const int64_t b = p.cu ? 0 : n;
    const T *pq = reinterpret_cast<const T *>(p.q.p) + b * p.q.batch + (int64_t)(h / p.q.div) * p.q.head;
    const T *pk = reinterpret_cast<const T *>(p.k.p) + b * p.k.batch + (int64_t)(h / p.k.div) * p.k.head;
    const T *pv = reinterpret_cast<const T *>(p.v.p) + b * p.v.batch + (int64_t)(h / p.v.div) * p.v.head;
    T *out = reinterpret_cast<T *>(p.out.p) + b * p.out.batch + (s.x + (int64_t)here.begin * kC) * p.out.token + (int64_t)h * p.out.head + v0 + 16 * mine + quad;
    pq += (s.x + (int64_t)here.begin * kC) * p.q.token;              // (these walk along: of the next chunk to be fetched)
    pk += (s.x + (int64_t)here.begin * kC) * p.k.token;
    pv += (s.x + (int64_t)here.begin * kC) * p.v.token;
    const float2 *pc = p.cum + ((int64_t)(s.z + here.begin) * p.heads + h) * kC;
    const int ms[2] = {half ? kM / 4 + (kM < 4) : 0, half ? kM / 2 : kM - 1};        // its tokens: of the four 16s the first and the last, or the others

    u32x4_t rq[kNk], rk[kNk], rv[kNv];
    float2 rc = make_float2(0.0f, 0.0f), re = rc;
    float decay = 0.0f;
    auto fetch = [&](int i) {
        const int len = min(kC, s.y - s.x - (here.begin + i) * kC);
#pragma unroll
        for (int j = 0; j < kNk; ++j) {
            const int at = tid + j * kLaThreads, row = at / kPerKey, d = at % kPerKey * kVec;
            rq[j] = load_piece<kFast>(pq, p.q.token, row, len, d, p.k.dim);
            rk[j] = load_piece<kFast>(pk, p.k.token, row, len, d, p.k.dim);
        }
#pragma unroll
        for (int j = 0; j < kNv; ++j) {
            const int at = tid + j * kLaThreads, row = at / kPerValue, d = at % kPerValue * kVec;
            rv[j] = load_piece<kFast>(pv, p.v.token, row, len, v0 + d, p.v.dim);
        }
        if (tid < kC) {
            if constexpr (kOwn) decay = p.decay && tid < len ? la_decay(p, b, s.x + (int64_t)(here.begin + i) * kC + tid, h) : 0.0f;
            else {
                rc = pc[tid];
                re = pc[kC - 1];
            }
        }
        pq += kC * p.q.token;
        pk += kC * p.k.token;
        pv += kC * p.v.token;
        pc += (int64_t)p.heads * kC;
    };
    if (here.count > 0) fetch(0);

    floatx4_t state[kHalf];                                          // key 16 (kHalf half + d) + quad + v, value v0 + 16 mine + col
    const int value = v0 + 16 * mine + col, key0 = 16 * kHalf * half;
    const int tiles_a = (p.k.dim + kLaTile - 1) / kLaTile;
    E *own = st + (16 * mine + col) * kPitchK + key0 + quad;         // its place as an operand
#pragma unroll
    for (int d = 0; d < kHalf; ++d) {
        const int at = kHalf * half + d;
        state[d] = floatx4_t{0, 0, 0, 0};
        if (!lone) {
            if (at / 4 < tiles_a)
                state[d] = *reinterpret_cast<const floatx4_t *>(w.local + (((int64_t)here.seg * p.heads + h) * tiles_a * tiles + here.tile * tiles_a + at / 4) * (kLaTile * kLaTile) +
                                                                mine * 4 * kBlock + 4 * (at % 4 * kWave + lane));
        } else if (w.from)
#pragma unroll
            for (int v = 0; v < 4; ++v)
                if (key0 + 16 * d + quad + v < p.k.dim && value < p.v.dim) state[d][v] = w.from[la_state_at(p, w, n, h, key0 + 16 * d + quad + v, value)];
    }
#pragma unroll
    for (int d = 0; d < kHalf; ++d) Op::put4(own + 16 * d, state[d]);
    bool carried = here.begin > 0 || w.from;                         // a state has come in
    const bool whole = p.k.dim == kKeys && p.v.dim - v0 >= kLaTile;  // the tiles' columns are all there
    for (int i = tid; i < kC * kPitchP; i += kLaThreads) pt[i] = E{};        // (behind the diagonal they stay)
    if (tid < 2) bad[tid] = 0;
    __syncthreads();
    for (int i = 0; i < here.count; ++i) {
        const int len = min(kC, s.y - s.x - (here.begin + i) * kC);
        bool none = false;
        if (len < kC || !whole) {
#pragma unroll
            for (int j = 0; j < kNk; ++j) {
                const int at = tid + j * kLaThreads, row = at / kPerKey, d = at % kPerKey * kVec;
                rq[j] = held_piece<kFast, T>(rq[j], row < len, d, p.k.dim);
                rk[j] = held_piece<kFast, T>(rk[j], row < len, d, p.k.dim);
            }
#pragma unroll
            for (int j = 0; j < kNv; ++j) {
                const int at = tid + j * kLaThreads, row = at / kPerValue, d = at % kPerValue * kVec;
                rv[j] = held_piece<kFast, T>(rv[j], row < len, v0 + d, p.v.dim);
            }
        }
#pragma unroll
        for (int j = 0; j < kNk; ++j) {
            const int at = tid + j * kLaThreads, row = at / kPerKey, d = at % kPerKey * kVec;
            if (kC * kPerKey % kLaThreads == 0 || row < kC) {
                put_piece<T, E>(qt + row * kPitchK + d, rq[j]);
                put_piece<T, E>(kt + row * kPitchK + d, rk[j]);
            }
        }
#pragma unroll
        for (int j = 0; j < kNv; ++j) {
            const int at = tid + j * kLaThreads, row = at / kPerValue, d = at % kPerValue * kVec;
            if (kC * kPerValue % kLaThreads == 0 || row < kC) put_piece<T, E>(vt + row * kPitchV + d, rv[j]);
            none |= piece_bad<T>(rv[j]);
        }
        if (none) bad[i & 1] = 1;
        if (tid < kC) {
            if constexpr (kOwn) {
                rc = la_sum_decays<kC>(decay, tid);
                re = make_float2(__shfl(rc.x, kC - 1, kC), __shfl(rc.y, kC - 1, kC));
            }
            cum[tid] = rc;
            if (kOwn && sizeof(E) == 4 && tid == 0) *kept = la_kept(re);
            weights[Op::place(tid)] = fast_exp2((re.x - rc.x) + (re.y - rc.y));
        }
        __syncthreads();
        if (i + 1 < here.count) fetch(i + 1);
        if (tid == 0) bad[(i + 1) & 1] = 0;

        // weights of the pairs, P[t][s]: tiles on and below the diagonal, the k-th of them in row tt, column ts
        for (int k = wave; k < kPairTiles; k += kLaWaves) {
            const int tt = k < 1 ? 0 : k < 3 ? 1 : k < 6 ? 2 : 3, ts = k - tt * (tt + 1) / 2, t = 16 * tt + col, r = 16 * ts + quad;
            floatx4_t acc = {0, 0, 0, 0};
#pragma unroll
            for (int k0 = 0; k0 < kKeys; k0 += Op::kStep)
                acc = Op::mma(Op::rows(kt, kPitchK, 16 * ts, k0, lane), Op::rows(qt, kPitchK, 16 * tt, k0, lane), acc);
            const float2 gt = cum[t];
#pragma unroll
            for (int v = 0; v < 4; ++v) {
                const float2 gs = cum[r + v];
                const float weight = acc[v] * fast_exp2((gt.x - gs.x) + (gt.y - gs.y));
                acc[v] = r + v <= t ? weight : 0.0f;
            }
            Op::put4_places(pt + t * kPitchP, r, acc);
        }
        floatx4_t acc[kHalfM];
        Frag values[kSteps];
        if (live) {
#pragma unroll
            for (int m = 0; m < kHalfM; ++m) acc[m] = floatx4_t{0, 0, 0, 0};
            if (carried) {
#pragma unroll
                for (int k0 = 0; k0 < kKeys; k0 += Op::kStep) {
                    const Frag a = Op::rows(st, kPitchK, 16 * mine, k0, lane);
#pragma unroll
                    for (int m = 0; m < kHalfM; ++m) acc[m] = Op::mma(a, Op::rows(qt, kPitchK, 16 * ms[m], k0, lane), acc[m]);
                }
#pragma unroll
                for (int m = 0; m < kHalfM; ++m) {
                    const float2 g = cum[16 * ms[m] + col];
                    acc[m] *= fast_exp2(g.x + g.y);
                }
            }
#pragma unroll
            for (int k = 0; k < kSteps; ++k) values[k] = Op::cols(vt, kPitchV, 16 * mine, k * Op::kStep, lane);
        }
        __syncthreads();
        if (live) {
            if (!bad[i & 1]) {
#pragma unroll
                for (int k = 0; k < kSteps; ++k)
#pragma unroll
                    for (int m = 0; m < kHalfM; ++m) acc[m] = Op::mma(values[k], Op::rows(pt, kPitchP, 16 * ms[m], k * Op::kStep, lane), acc[m]);
            } else {
                const int t = la_here(col), d = la_here(16 * mine + quad);
#pragma unroll
                for (int m = 0; m < kHalfM; ++m)
                    for (int r = 0; r <= 16 * ms[m] + t; ++r) {
                        const float weight = to_f32(pt[(16 * ms[m] + t) * kPitchP + Op::place(r)]);
#pragma unroll
                        for (int v = 0; v < 4; ++v) acc[m][v] += weight * to_f32(vt[r * kPitchV + d + v]);
                    }
            }
#pragma unroll
            for (int m = 0; m < kHalfM; ++m) {
                const int t = 16 * ms[m] + col;
                if (t < len) store4(out + (int64_t)t * p.out.token, acc[m] * p.scale, p.v.dim - value + col - quad);
            }
            if (i + 1 < here.count || (last && w.to)) {              // somebody wants the state behind this chunk
                LaKeep<E> keep;
                keep.set(cum[kC - 1], kOwn ? kept : p.kept + (int64_t)(s.z + here.begin + i) * p.heads + h);
#pragma unroll
                for (int d = 0; d < kHalf; ++d) keep.scale(state[d]);
#pragma unroll
                for (int k = 0; k < kSteps; ++k) {
                    Frag parts[kParts], keys[kHalf];
                    Op::template weigh<kParts>(values[k], weights + k * Op::kStep, lane, parts);
#pragma unroll
                    for (int d = 0; d < kHalf; ++d) keys[d] = Op::cols(kt, kPitchK, key0 + 16 * d, k * Op::kStep, lane);
#pragma unroll
                    for (int q = 0; q < kParts; ++q)
#pragma unroll
                        for (int d = 0; d < kHalf; ++d) state[d] = Op::mma(keys[d], parts[q], state[d]);
                }
#pragma unroll
                for (int d = 0; d < kHalf; ++d) Op::put4(own + 16 * d, state[d]);
            }
        }
        out += kC * p.out.token;
        carried = true;
        __syncthreads();
    }
    if (!w.to || !last) return;
#pragma unroll
    for (int d = 0; d < kHalf; ++d)
#pragma unroll
        for (int v = 0; v < 4; ++v)
            if (key0 + 16 * d + quad + v < p.k.dim && value < p.v.dim) w.to[la_state_at(p, w, n, h, key0 + 16 * d + quad + v, value)] = state[d][v];
}

// ---- host ----------------------------------------------------------------------------------------------------------------------------
// Segments: where the sequences alone do not give the chip its workgroups (`tiles` for a head), each is cut so that there are two to a CU, into
// `shortest` chunks at least: a segment is walked twice.  192 workgroups are enough, since the cut costs two launches and the second reading; 128 where
// chains are short.  us cut / whole, heads of 64, bf16, forward: 128 workgroups of 8 chunks 32 / 27, of 16 42 / 44, of 25 55 / 63, of 64 101 / 140; 192 of 8 42 / 27, of 25 78 / 62,
// of 64 168 / 148.  A training step whose walks for the gradients are cut or whole: 192 of 16 139 / 130, of 25 177 / 173, of 32 220 / 218, of 64 416 / 423; 256 of 64
// 522 / 502; in single precision 192 of 25 200 / 191, of 32 263 / 262, of 64 479 / 486.  So the border is right up to 32 chunks and 2 % off at 64.
constexpr int kLaWhole = 5;          // chunks of a sequence that is never cut
int la_plan(LaArgs &p, int chunk, int64_t tiles, int shortest, int lanes) {
    // Places of tokens are 32-bit numbers on the GPU, those of whole chunks too; the table of packed sequences' chunks runs on behind the last token by a chunk
    // for each sequence and two (la_find_chunk).
    if (p.tokens + ((p.cu ? (int64_t)p.n_seqs : 0) + 3) * chunk > 0x7fffffff) return SS2D_ENOTSUP;
    const int64_t per_seq = ((int64_t)p.tokens + chunk - 1) / chunk, alone = (int64_t)p.n_seqs * p.heads * tiles;
    const int64_t want = alone >= 192 || (alone >= 128 && per_seq <= 16) ? 1 : (512 + p.heads * tiles - 1) / (p.heads * tiles);
    int64_t chunks, segs, seg_chunks;
    if (p.cu) {
        chunks = (int64_t)p.tokens / chunk + p.n_seqs + 2;
        // Whatever the longest of them is.  As if all tokens were one sequence, three times the workgroups that are there at once, since most of the segments are
        // shorter than that, and five chunks at least; against half of the workgroups and two chunks, prompts / training: 12 011 tokens in 16 sequences, 24 heads of
        // 128 x 64, bf16, 148 -> 139 / 659 -> 628 us; 30 000 in 4, 16 heads of 128, 291 -> 283 / 1525 -> 1263; 8192 in 40, 32 heads of 64, 105 -> 107 / 369 -> 378.
        seg_chunks = (per_seq * p.heads * tiles + 1535) / 1536;
        seg_chunks = seg_chunks < kLaWhole ? kLaWhole : seg_chunks;
        segs = per_seq <= seg_chunks ? p.n_seqs : chunks / seg_chunks + p.n_seqs;
    } else {
        chunks = per_seq * p.n_seqs;
        const int64_t each = (want + p.n_seqs - 1) / p.n_seqs;
        seg_chunks = (per_seq + each - 1) / each;
        // (a few chunks take less than the two launches that cutting them takes: 300 tokens, 8 heads of 64, bf16, 20.0 -> 18.8 us, training 60 -> 53)
        seg_chunks = per_seq <= kLaWhole ? kLaWhole : seg_chunks < shortest ? shortest : seg_chunks;
        p.segs_per_seq = per_seq <= seg_chunks ? 1 : (int)((per_seq + seg_chunks - 1) / seg_chunks);
        segs = (int64_t)p.segs_per_seq * p.n_seqs;
    }
    if (chunks > kLaLaunch / lanes / p.heads || segs > kLaLaunch / kLaThreads / p.heads / la_tiles(p)) return SS2D_ENOTSUP;
    p.per_seq = (int)per_seq;
    p.max_chunks = (int)chunks;
    p.seg_chunks = (int)seg_chunks;
    p.max_segs = (int)segs;
    return SS2D_OK;
}

int la_tables(const LaArgs &p, int chunk, int out_bytes, void *stream) {
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    if (p.cu) la_sequences_kernel<<<1, kBlock, 0, st>>>(p, chunk);
    const int64_t total = (int64_t)p.max_chunks * p.heads;
    if (total == 0) return launch_status();
    const int64_t per = kBlock / chunk, grid = (total + per - 1) / per;
    auto go = [&](auto kernel) { kernel<<<(uint32_t)grid, kBlock, 0, st>>>(p, total); };
    const bool clear = p.cu && out_bytes > 0;
    if (chunk == 64) clear ? go(la_chunks_kernel<64, 2>) : go(la_chunks_kernel<64, 0>);          // (bf16)
    else if (clear) out_bytes == 2 ? go(la_chunks_kernel<32, 2>) : go(la_chunks_kernel<32, 4>);
    else go(la_chunks_kernel<32, 0>);
    return launch_status();
}

template <typename Op, typename T> static int la_forward(const LaArgs &p, void *stream) {
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    int rc = SS2D_OK;
    const bool own = !p.cu && p.per_seq <= kLaOwnChunks && p.k.dim <= kLaOwnKeys && p.max_segs <= p.n_seqs;
    if (!own && (rc = la_tables(p, Op::kChunk, (int)sizeof(T), stream)) != SS2D_OK) return rc;
    LaWalk w = {};
    w.a = p.k; w.b = p.v;
    w.from = p.initial; w.to = p.final;
    w.from_a = p.v.dim; w.from_b = 1;
    w.local = p.local;
    w.exact = p.final != nullptr;
    if ((rc = la_segments<Op, T>(p, &w, 1, st)) != SS2D_OK) return rc;
    const uint32_t total = (uint32_t)((int64_t)p.max_segs * p.heads * ((p.v.dim + kLaTile - 1) / kLaTile));
    auto go = [&](auto kernel, int keys) {
        constexpr int c = Op::kChunk;
        const size_t bytes = sizeof(typename Op::E) * ((2 * c + kLaTile) * (keys + Op::kPad) + c * (kLaTile + Op::kPad + c + Op::kPad)) + c * (sizeof(float) + sizeof(float2)) + 16;
        kernel<<<total, kLaThreads, bytes, st>>>(p, w, total);       // (up to 146 KB of LDS: this runtime asks for no attribute above 64)
    };
    const bool fast = p.q.pieces && p.k.pieces && p.v.pieces;
    auto sized = [&](auto tiles) {
        constexpr int kTiles = decltype(tiles)::value, kMost = Op::kMostParts, kLess = kMost < 2 ? kMost : 2;
        auto parted = [&](auto own_sums) {
            constexpr bool kOwn = decltype(own_sums)::value;
            if (w.exact) fast ? go(la_out_kernel<Op, T, kTiles, kMost, true, kOwn>, 16 * kTiles) : go(la_out_kernel<Op, T, kTiles, kMost, false, kOwn>, 16 * kTiles);
            else fast ? go(la_out_kernel<Op, T, kTiles, kLess, true, kOwn>, 16 * kTiles) : go(la_out_kernel<Op, T, kTiles, kLess, false, kOwn>, 16 * kTiles);
        };
        if constexpr (16 * kTiles <= kLaOwnKeys)
            if (own) return parted(std::true_type{});
        parted(std::false_type{});
    };
    if (p.k.dim <= 32) sized(std::integral_constant<int, 2>{});
    else if (p.k.dim <= 64) sized(std::integral_constant<int, 4>{});
    else if (p.k.dim <= 128) sized(std::integral_constant<int, 8>{});
    else sized(std::integral_constant<int, 16>{});
    return launch_status();
}

LaSide la_side(const void *ptr, int64_t batch, int64_t token, int64_t head, int heads, int own_heads, int dim, int size) {
    LaSide s = {};
    s.p = const_cast<void *>(ptr);
    s.batch = batch; s.token = token; s.head = head;
    s.div = own_heads > 0 ? heads / own_heads : 1;
    s.dim = dim;
    s.pieces = dim * size >= 16 && token >= 0 && token * size < (1 << 24);
    return s;
}

int la_chunk(int dtype) { return dtype == SS2D_BF16 ? OperandBf16::kChunk : OperandF32::kChunk; }

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
    a.q = la_side(p->q, p->q_batch_stride, p->q_token_stride, p->q_head_stride, p->heads, p->q_heads, p->key_dim, size);
    a.k = la_side(p->k, p->k_batch_stride, p->k_token_stride, p->k_head_stride, p->heads, p->k_heads, p->key_dim, size);
    a.v = la_side(p->v, p->v_batch_stride, p->v_token_stride, p->v_head_stride, p->heads, p->v_heads, p->value_dim, size);
    const int64_t row = (int64_t)p->heads * p->value_dim;
    a.out = la_side(p->out, row * p->seqlen, row, p->value_dim, p->heads, p->heads, p->value_dim, size);
    if (a.heads == 0 || a.n_seqs == 0) { empty = true; return SS2D_OK; }
    const bool rows = a.tokens > 0;
    if (rows && (!p->q || !p->k || !p->v)) return SS2D_EINVAL;
    return SS2D_OK;
}

static int la_forward_plan(const ss2d_linear_attention_params *p, LaArgs &a, bool &empty) {
    const int rc = la_arguments(p, a, empty);
    return rc != SS2D_OK || empty ? rc : la_plan(a, la_chunk(p->dtype), (a.v.dim + kLaTile - 1) / kLaTile, 2, la_chunk(p->dtype));
}

static int64_t la_round(int64_t n) { return (n + 255) / 256 * 256; }

// Lays a call's workspace out from `base` on and says how long it is.  low: what the rounding of states leaves is kept.
int64_t la_carve(LaArgs &p, int dtype, char *base, bool backward, bool low) {
    const int chunk = la_chunk(dtype), size = dtype == SS2D_BF16 ? 2 : 4;
    const int64_t entries = (int64_t)p.max_chunks * p.heads, state = (int64_t)la_state_dim(p.k.dim) * la_state_dim(p.v.dim);
    const int64_t tiles = la_tiles(p);
    int64_t at = 0;
    auto take = [&](auto *&ptr, int64_t bytes) {
        ptr = reinterpret_cast<std::remove_reference_t<decltype(ptr)>>(base + at);
        at += la_round(bytes);
    };
    take(p.chunks, sizeof(int4) * (int64_t)p.max_chunks);
    take(p.seqs, p.cu ? sizeof(int4) * ((int64_t)p.n_seqs + 1) : 0);
    take(p.cum, sizeof(float2) * entries * chunk);
    take(p.kept, sizeof(float2) * entries);
    p.low = low ? entries * state : 0;
    if (backward) {
        take(p.states, (low ? 3 : 1) * size * entries * state);
        take(p.dstates, (low ? 3 : 1) * size * entries * state);
        take(p.dstates_t, la_turned(p, dtype) ? size * entries * state : 0);
    }
    p.local_floats = p.max_segs > p.n_seqs ? (la_round(4 * (int64_t)p.max_segs * p.heads * (tiles * kLaTile * kLaTile + 1)) / 4) : 0;
    take(p.local, 4 * p.local_floats * (backward ? 2 : 1));
    return at < 256 ? 256 : at;                                      // (a caller has an address to give)
}

}  // namespace ss2d

using namespace ss2d;

extern "C" int64_t ss2d_linear_attention_workspace_bytes(const ss2d_linear_attention_params *params) {
    LaArgs a;
    bool empty;
    const int rc = la_forward_plan(params, a, empty);
    if (rc != SS2D_OK || empty) return rc;
    return la_carve(a, params->dtype, nullptr, false, false);
}

extern "C" int ss2d_linear_attention_fwd(const ss2d_linear_attention_params *params, void *workspace, int64_t workspace_bytes, void *stream) {
    LaArgs a;
    bool empty;
    const int rc = la_forward_plan(params, a, empty);
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
