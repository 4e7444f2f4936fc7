// kV neighbouring values of a row as one load or store, at any address of their type (1: by themselves).  Stores go past the caches: what is written is not read again by
// its launch, and what is read is left more room (a training step of 8 x 4096 tokens' convolution 156 -> 139 us, a norm of 32 maps of 56 x 56 29 -> 25; loads of
// that kind cost what the stores gain).
#pragma once
#include "ss2d_common.h"

namespace ss2d {

template <typename T, int kV> struct RowPiece {
    static constexpr int kWords = kV * (int)sizeof(T) / 4 > 0 ? kV * (int)sizeof(T) / 4 : 1;
    uint32_t w[kWords];
    __device__ __forceinline__ float get(int i) const {
        if constexpr (sizeof(T) == 4) return bits_to_f32(w[i]);
        else return i & 1 ? unpack_hi<T>(w[i / 2]) : unpack_lo<T>(w[i / 2]);
    }
};

template <typename T, int kV> __device__ __forceinline__ RowPiece<T, kV> load_row_piece(const T *p) {
    RowPiece<T, kV> r;
    if constexpr (kV == 1) {
        if constexpr (sizeof(T) == 4) r.w[0] = f32_to_bits(*p);
        else r.w[0] = p->bits;
    } else {
        constexpr int kWords = RowPiece<T, kV>::kWords;
        typedef uint32_t here __attribute__((ext_vector_type(kWords), aligned(sizeof(T))));
        const here v = *reinterpret_cast<const here *>(p);
#pragma unroll
        for (int i = 0; i < kWords; ++i) r.w[i] = v[i];
    }
    return r;
}

template <typename T, int kV> __device__ __forceinline__ void store_row_piece(T *p, const float (&v)[kV]) {
    if constexpr (kV == 1) {
        *p = from_f32<T>(v[0]);
    } else {
        constexpr int kWords = RowPiece<T, kV>::kWords;
        typedef uint32_t here __attribute__((ext_vector_type(kWords), aligned(sizeof(T))));
        here w;
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
            if constexpr (sizeof(T) == 4) w[i] = f32_to_bits(v[i]);
            else w[i] = pack2_from_f32<T>(v[2 * i], v[2 * i + 1]);
        }
        __builtin_nontemporal_store(w, reinterpret_cast<here *>(p));
    }
}

}  // namespace ss2d
