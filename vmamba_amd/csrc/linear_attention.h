// Linear attention with a decay for each head, what its kernels share: per head a state S of Dk x Dv values,
//     S_t = exp(g_t) S_(t-1) + k_t v_t^T,   o_t = scale q_t^T S_t
// -- the selective scan with a matrix for a state and one decay for all of it, which makes its products matrix products.  A sequence
// is cut into chunks of C tokens.  With G_t the sum of the chunk's g up to and with t, and S the state before the chunk,
//     o_t = scale sum_(s <= t) exp(G_t - G_s) (q_t . k_s) v_s + scale exp(G_t) q_t^T S,
//     S after = exp(G_C) S + sum_s exp(G_C - G_s) k_s v_s^T,
// so what goes from chunk to chunk is the state alone.  Outputs and states are one walk over a sequence's chunks (linear_attention.hip); for the gradients two
// walks store the states before and behind every chunk, and the chunks are then independent of one another (linear_attention_bwd.hip).  Everything that is a sum of g stands as a pair of floats from a sum in 64 bits and
// goes through exp as a difference first: a decay of -inf (a reset) or a long sum loses nothing.
//
// Operands.  bf16 goes to the 16-bit matrix cores as it is; what is computed on the way (weights of pairs, states) is rounded to bf16
// where it becomes an operand of a product that is itself rounded to bf16 at its end, and split into two bf16 values, three where its
// result is kept in 32 bits (states, single precision decays' gradients).  fp16 and fp32 go to the fp32 matrix cores: the states' and
// weights' range is not fp16's.  Chunks are 64 tokens in bf16, two steps of 32 of its matrix instruction, and 32 on the fp32 cores, where the
// pairs' share of the work is dear (153 TFLOP/s against 1129).
#pragma once
#include "ss2d_common.h"

namespace ss2d {

constexpr int kLaMaxDim = 256;       // of a key or value
constexpr int kLaTile = 64;          // sides of the piece of a state that a workgroup walks
constexpr int kLaThreads = 512;      // of the largest workgroups
constexpr int64_t kLaLaunch = 0xffffffff;                            // threads of a launch
constexpr float kLog2e = 1.4426950408889634f;

struct LaSide {                      // q, k, v, out or a gradient: (batch, token, head, dim), the last one dense
    void *p;
    int64_t batch, token, head;      // strides in elements
    int32_t div;                     // heads of the state to one of this
    int32_t dim;
    int32_t pieces;                  // what is read: heads of a piece of 16 bytes at least, tokens at strides below 2^24 bytes
};

struct LaArgs {
    LaSide q, k, v, out, dout, dq, dk, dv;
    const void *decay;               // (batch, token, head) or (head) or NULL
    void *ddecay;
    int64_t decay_batch, decay_token, decay_head;
    int32_t decay_dtype, ddecay_f32;
    const int32_t *cu;               // packed sequences: n_seqs + 1 places, or NULL
    int32_t batch, tokens, heads, n_seqs;
    int32_t per_seq;                 // chunks of a sequence that is not packed
    int32_t max_chunks, seg_chunks, max_segs, segs_per_seq;
    float scale;
    const float *initial, *dfinal;   // (n_seqs, heads, Dk, Dv), dense
    float *final, *dinitial;
    // workspace
    int4 *chunks;                    // {batch, first token, tokens, sequence}; no tokens: unused; sequence -1: rows of no sequence
    int4 *seqs;                      // packed: {start, end, first chunk, first segment}, and {rows before, rows' end, chunks, segments} behind them
    float2 *cum;                     // [chunk][head][C]: G in log2 units, high and low part
    float2 *kept;                    // [chunk][head]: exp of the whole chunk's sum, high and low part
    void *states, *dstates, *dstates_t;
    int64_t low;                     // elements from a state's bf16 value to what its rounding left, and on to what that one's left; 0: not kept
    float *local;                    // [segment][head][tile][4096] and behind it [segment][head] decays; for the backward twice
    int64_t local_floats;
};

// ---- operands of the matrix cores --------------------------------------------------------------------------------------------
// rows(): the lane's part of 16 rows of a tile that is dense along the sum (k); cols(): of 16 columns of a tile that is dense across it.
// A lane holds the same k for A and B, so the order inside a step is free.
struct OperandF32 {
    using E = float;
    using Frag = floatx4_t;
    static constexpr int kStep = 16, kChunk = 32, kPad = 4;
    static __device__ __forceinline__ Frag rows(const E *tile, int pitch, int row0, int k0, int lane) {
        return *reinterpret_cast<const Frag *>(tile + (row0 + (lane & 15)) * pitch + k0 + 4 * (lane >> 4));
    }
    static __device__ __forceinline__ Frag cols(const E *tile, int pitch, int col0, int k0, int lane) {
        const E *p = tile + (k0 + 4 * (lane >> 4)) * pitch + col0 + (lane & 15);
        return Frag{p[0], p[pitch], p[2 * pitch], p[3 * pitch]};
    }
    static __device__ __forceinline__ floatx4_t mma(Frag a, Frag b, floatx4_t c) {
#pragma unroll
        for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], c, 0, 0, 0);
        return c;
    }
    static __device__ __forceinline__ void put4(E *p, floatx4_t v) { *reinterpret_cast<floatx4_t *>(p) = v; }
    // Where a product sums over rows of a tile (cols()), what rows() reads against it stands in cols()'s order of k: place() of k inside the row,
    // put4_places() four neighbours from a multiple of 4 on.
    static __device__ __forceinline__ int place(int k) { return k; }
    static __device__ __forceinline__ void put4_places(E *row, int k, floatx4_t v) { put4(row + k, v); }
    static __device__ __forceinline__ Frag in_places(Frag f) { return f; }          // of rows() that stand as they are
    // The operand's values times their tokens' weights (weight: of token k0 on, in places), in kParts operands whose sum it is
    static constexpr int kMostParts = 1;
    template <int kParts> static __device__ __forceinline__ void weigh(Frag f, const float *weight, int lane, Frag (&parts)[kParts]) {
        parts[0] = f * *reinterpret_cast<const floatx4_t *>(weight + 4 * (lane >> 4));
    }
};

struct OperandBf16 {
    using E = bf16_t;
    using Frag = u32x4_t;
    static constexpr int kStep = 32, kChunk = 64, kPad = 8;
    static __device__ __forceinline__ Frag rows(const E *tile, int pitch, int row0, int k0, int lane) {
        return *reinterpret_cast<const Frag *>(tile + (row0 + (lane & 15)) * pitch + k0 + 8 * (lane >> 4));
    }
    // ds_read_b64_tr_b16: of the four rows that a group of 16 lanes names, 8 bytes to a lane, a lane gets its column.  A group takes the even rows of
    // eight, then the odd ones: at these tiles' pitches (36 and 68 dwords, modulo 64) four neighbouring rows would share banks.
    static __device__ __forceinline__ Frag cols(const E *tile, int pitch, int col0, int k0, int lane) {
        typedef short s16x4 __attribute__((ext_vector_type(4)));
        typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
        using Lds = __attribute__((address_space(3))) s16x4;
        const E *p = tile + (k0 + 8 * (lane >> 4) + 2 * ((lane & 15) >> 2)) * pitch + col0 + 4 * (lane & 3);
        const u32x2 lo = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds *)p));
        const u32x2 hi = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds *)(p + pitch)));
        return Frag{lo[0], lo[1], hi[0], hi[1]};
    }
    static __device__ __forceinline__ int place(int k) { return (k & ~7) + 4 * (k & 1) + ((k & 7) >> 1); }
    static __device__ __forceinline__ void put4_places(E *row, int k, floatx4_t v) {
        uint32_t *p = reinterpret_cast<uint32_t *>(row + (k & ~7) + ((k & 4) >> 1));
        p[0] = pack2_from_f32<bf16_t>(v[0], v[2]);
        p[2] = pack2_from_f32<bf16_t>(v[1], v[3]);
    }
    static __device__ __forceinline__ Frag in_places(Frag f) {
        constexpr uint32_t kLow = 0x05040100u, kHigh = 0x07060302u;  // of two dwords the low halves, the high ones
        return Frag{__builtin_amdgcn_perm(f[1], f[0], kLow), __builtin_amdgcn_perm(f[3], f[2], kLow), __builtin_amdgcn_perm(f[1], f[0], kHigh),
                    __builtin_amdgcn_perm(f[3], f[2], kHigh)};
    }
    static __device__ __forceinline__ floatx4_t mma(Frag a, Frag b, floatx4_t c) { return mfma_16x16x32(bf16_t{}, a, b, c); }
    static __device__ __forceinline__ void put4(E *p, floatx4_t v) {
        *reinterpret_cast<uint2 *>(p) = make_uint2(pack2_from_f32<bf16_t>(v[0], v[1]), pack2_from_f32<bf16_t>(v[2], v[3]));
    }
    // (bf16 of the value, of what that left, and of what that left: 24 bits.  Of an infinity it is NaN that is left: a state with one is of no use.)
    static constexpr int kMostParts = 3;
    template <int kParts> static __device__ __forceinline__ void weigh(Frag f, const float *weight, int lane, Frag (&parts)[kParts]) {
        const floatx4_t w[2] = {*reinterpret_cast<const floatx4_t *>(weight + 8 * (lane >> 4)), *reinterpret_cast<const floatx4_t *>(weight + 8 * (lane >> 4) + 4)};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float x = unpack_lo<bf16_t>(f[i]) * w[i / 2][2 * i % 4], y = unpack_hi<bf16_t>(f[i]) * w[i / 2][2 * i % 4 + 1];
#pragma unroll
            for (int k = 0; k < kParts; ++k) {
                parts[k][i] = pack2_from_f32<bf16_t>(x, y);
                if (k + 1 == kParts) break;
                x -= unpack_lo<bf16_t>(parts[k][i]);
                y -= unpack_hi<bf16_t>(parts[k][i]);
            }
        }
    }
};

// ---- tiles ------------------------------------------------------------------------------------------------------------------------
template <typename T> constexpr int kVecOf = 16 / (int)sizeof(T);

// 16 bytes' worth of row `row` of `rows` (one at least), from column c on, c a multiple of a piece.  kFast: rows hold a piece at least and a chunk's offsets
// fit 32 bits; the load is then unconditional, wherever it begins -- a row or column that is not there repeats another, the last piece is the one that ends
// with its row -- so that nothing waits for it before it is used, and held_piece() puts it in its place and makes zeros of what is not there.  Otherwise
// element by element.  (8 x 4096 tokens, 16 heads of 127 in bf16, the outputs alone: 248 us, element by element 634; of 128, one value off the 16-byte grid, 221 and 641,
// on it 208.  With the final state 264 and 253.)
template <bool kFast, typename T> __device__ __forceinline__ u32x4_t load_piece(const T *base, int64_t stride, int row, int rows, int c, int cols) {
    if constexpr (kFast) {
        typedef uint32_t here __attribute__((ext_vector_type(4), aligned(2)));
        const uint32_t at = (uint32_t)min(row, rows - 1) * (uint32_t)stride + (uint32_t)min(c, cols - kVecOf<T>);
        return *reinterpret_cast<const here *>(reinterpret_cast<const char *>(base) + at * (uint32_t)sizeof(T));
    }
    union { T e[kVecOf<T>]; u32x4_t w; } u;
    u.w = u32x4_t{0, 0, 0, 0};
    if (row < rows)
#pragma unroll
        for (int i = 0; i < kVecOf<T>; ++i)
            if (c + i < cols) u.e[i] = base[row * stride + c + i];
    return u.w;
}
template <bool kFast, typename T> __device__ __forceinline__ u32x4_t held_piece(u32x4_t piece, bool in, int c, int cols) {
    if constexpr (kFast) {
        if (cols % kVecOf<T> != 0) {                                 // the last piece: its first values are those that end the one before
            const int bytes = max(c + kVecOf<T> - cols, 0) * (int)sizeof(T);
            if (bytes & 8) piece = u32x4_t{piece[2], piece[3], 0, 0};
            if (bytes & 4) piece = u32x4_t{piece[1], piece[2], piece[3], 0};
            if (sizeof(T) == 2 && bytes & 2)
                piece = u32x4_t{__builtin_amdgcn_alignbit(piece[1], piece[0], 16), __builtin_amdgcn_alignbit(piece[2], piece[1], 16), __builtin_amdgcn_alignbit(piece[3], piece[2], 16),
                                piece[3] >> 16};
        }
        in = in && c < cols;
#pragma unroll
        for (int i = 0; i < 4; ++i) piece[i] = in ? piece[i] : 0u;
    }
    return piece;
}

template <typename T> __device__ __forceinline__ float piece_at(u32x4_t w, int i) {
    if constexpr (sizeof(T) == 4) return bits_to_f32(w[i]);
    else return i % 2 ? unpack_hi<T>(w[i / 2]) : unpack_lo<T>(w[i / 2]);
}

// Whether one of the piece's values is infinite or NaN
template <typename T> __device__ __forceinline__ bool piece_bad(u32x4_t w) {
    bool bad = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 4) bad |= (w[i] & 0x7f800000u) == 0x7f800000u;
        else {
            constexpr uint32_t m = __is_same(T, bf16_t) ? 0x7f80u : 0x7c00u;
            bad |= (w[i] & m) == m || (w[i] & (m << 16)) == (m << 16);
        }
    }
    return bad;
}

template <typename T, typename E> __device__ __forceinline__ void put_piece(E *lds, u32x4_t w) {
    if constexpr (sizeof(T) == sizeof(E)) *reinterpret_cast<u32x4_t *>(lds) = w;
    else {
#pragma unroll
        for (int i = 0; i < kVecOf<T>; i += 4)
            *reinterpret_cast<floatx4_t *>(lds + i) = floatx4_t{piece_at<T>(w, i), piece_at<T>(w, i + 1), piece_at<T>(w, i + 2), piece_at<T>(w, i + 3)};
    }
}

// Four neighbouring results of one token to memory, wherever they begin, `left` of them inside the row
template <typename T> __device__ __forceinline__ void store4(T *p, floatx4_t v, int left) {
    typedef float four __attribute__((ext_vector_type(4), aligned(4)));
    typedef uint32_t two __attribute__((ext_vector_type(2), aligned(2)));
    if (left >= 4) {
        if constexpr (sizeof(T) == 4) *reinterpret_cast<four *>(p) = four{v[0], v[1], v[2], v[3]};
        else *reinterpret_cast<two *>(p) = two{pack2_from_f32<T>(v[0], v[1]), pack2_from_f32<T>(v[2], v[3])};
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (i < left) p[i] = from_f32<T>(v[i]);
}

// The value, as if it were made here: what follows from it is not computed ahead of a branch that is hardly ever taken
__device__ __forceinline__ int la_here(int x) {
    asm volatile("" : "+v"(x));
    return x;
}

__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }            // (what is below 2^-126 is 0)

// What a chunk leaves of the state that it finds.  It is multiplied in chunk after chunk, and where a head's decay is learnt all of them are alike and so is
// what rounding does to them: in single precision it is a pair of floats.
__device__ __forceinline__ float2 la_kept(float2 end) {
    const double keep = exp2((double)end.x + (double)end.y);
    const float high = (float)keep;
    return make_float2(high, (float)(keep - (double)high));
}
template <typename E> struct LaKeep {
    float high, low;
    // of a chunk that ends with the sum `end` and whose pair stands at *kept
    __device__ __forceinline__ void set(float2 end, const float2 *kept) {
        if constexpr (sizeof(E) == 4) {
            high = kept->x;
            low = kept->y;
        } else high = fast_exp2(end.x + end.y);
    }
    __device__ __forceinline__ float of(float v) const {
        if constexpr (sizeof(E) == 4) return fmaf(v, high, v * low);
        return v * high;
    }
    __device__ __forceinline__ void scale(floatx4_t &v) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = of(v[i]);
    }
    __device__ __forceinline__ void add(floatx4_t &v, floatx4_t more) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = fmaf(v[i], high, fmaf(v[i], low, more[i]));
    }
};

inline __host__ __device__ int la_up(int n, int m) { return (n + m - 1) / m * m; }
// Rows of a state stand at a pitch that every operand's step divides, with zeros behind them
inline __host__ __device__ int la_state_dim(int d) { return la_up(d, 32); }

__device__ __forceinline__ float load_decay(const void *p, int64_t at, int dtype) {
    return dtype == SS2D_F32 ? reinterpret_cast<const float *>(p)[at] : dtype == SS2D_BF16 ? to_f32(reinterpret_cast<const bf16_t *>(p)[at])
                                                                                          : to_f32(reinterpret_cast<const f16_t *>(p)[at]);
}

// Whether the gradients read the states behind the chunks (E) in both orders from memory: of bf16 heads up to 128 they turn them in LDS
constexpr int kLaTurnDim = 128;
inline bool la_turned(const LaArgs &p, int dtype) { return dtype != SS2D_BF16 || p.k.dim > kLaTurnDim || p.v.dim > kLaTurnDim; }

// A sequence's {start, end, first chunk, first segment}, whichever way the sequences stand
__device__ __forceinline__ int4 la_sequence(const LaArgs &p, int n) {
    return p.cu ? p.seqs[n] : make_int4(0, p.tokens, n * p.per_seq, n * p.segs_per_seq);
}

// The walks over the states that linear_attention.hip offers to both directions: a and b are (k, v), (v, k), (do, q)
struct LaWalk {
    LaSide a, b;                     // M = sum of w a b^T, stored as rows of b's dimension, dense in a's
    void *out, *out_t;               // [chunk][head][Db][Da] and, where wanted, [chunk][head][Da][Db]
    const float *from;               // the state to begin with, element (ia, ib) at ia * from_a + ib * from_b; NULL: zero
    float *to;                       // the state to end with, or NULL
    float *local;                    // as LaArgs::local
    int64_t low;                     // as LaArgs::low, of out
    int32_t from_a, from_b;
    int32_t reverse;                 // from the last chunk to the first, weights scale exp(G_t) instead of exp(G_C - G_s)
    int32_t exact;                   // the states are kept in 32 bits: three parts to a weighted 16-bit operand instead of two
};
// Sizes of the tables and segments, for `tiles` workgroups a head; a launch takes `lanes` threads for each chunk and head.
int la_plan(LaArgs &p, int chunk, int64_t tiles, int shortest, int lanes);
int la_tables(const LaArgs &p, int chunk, int out_bytes, void *stream);                // chunks, seqs, cum and kept; out_bytes: of a value of p.out, to clear its rows of no sequence, or 0
template <typename Op, typename T> int la_walks(const LaArgs &p, const LaWalk *w, int n, void *stream);        // states before all chunks, one walk or two side by side
}  // namespace ss2d
