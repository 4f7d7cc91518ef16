// few_rows.h -- products of a few rows with a large matrix, bound by reading the matrix once: 16 rows of it by up
// to 16 rows of x in a workgroup, operands of the MFMA straight from memory.
//
// A round is 128 bytes of each row: lane (i = lane & 15, g = lane >> 4) holds bytes 32 g .. 32 g + 31 of its row of
// the matrix and of its row of x, two 16-byte pieces.  Which values of the contraction an MFMA step takes is free
// as long as both operands agree, so every row is read in whole lines.  The waves take every WAVES-th round.
#pragma once

#include "tile_gemm.h"

namespace few {

using namespace tile;

constexpr int WAVES = 4, THREADS = 64 * WAVES, UNROLL = 4;

template <class T> __device__ __forceinline__ typename T::acc piece(u32x4 a, u32x4 b, typename T::acc c)
{
    if constexpr (std::is_same<T, F32>::value) {     // float32 on its own MFMA: the weights' bytes are the bound here
        const f32x4 fa = __builtin_bit_cast(f32x4, a), fb = __builtin_bit_cast(f32x4, b);
#pragma unroll
        for (int k = 0; k < 4; ++k) c = __builtin_amdgcn_mfma_f32_16x16x4f32(fa[k], fb[k], c, 0, 0, 0);
        return c;
    } else {
        return T::mma(a, b, c);
    }
}

// this wave's share of the products of matrix row w (i = lane & 15: four consecutive rows of the result per lane)
// with row x; rows that do not exist are given as any that do
template <class T>
__device__ __forceinline__ typename T::acc dot(const typename T::elem *w, const typename T::elem *wend, const typename T::elem *x,
                                               const typename T::elem *xend, int K)
{
    typedef typename T::elem E;
    constexpr int ROUND = 128 / sizeof(E), PIECE = 16 / sizeof(E);
    const int g = (threadIdx.x & 63) >> 4, wave = threadIdx.x >> 6;
    typename T::acc acc = {0, 0, 0, 0};
    const int rounds = K / ROUND;
    w += g * 2 * PIECE;
    x += g * 2 * PIECE;
    int r = wave;
    for (; r + (UNROLL - 1) * WAVES < rounds; r += UNROLL * WAVES) {
        u32x4 a[UNROLL][2], b[UNROLL][2];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                a[u][h] = *reinterpret_cast<const u32x4u *>(w + (r + u * WAVES) * ROUND + h * PIECE);
                b[u][h] = *reinterpret_cast<const u32x4u *>(x + (r + u * WAVES) * ROUND + h * PIECE);
            }
#pragma unroll
        for (int u = 0; u < UNROLL; ++u)
#pragma unroll
            for (int h = 0; h < 2; ++h) acc = piece<T>(a[u][h], b[u][h], acc);
    }
    for (; r * ROUND < K; r += WAVES) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int c = r * ROUND + h * PIECE, left = K - c - g * 2 * PIECE;
            acc = piece<T>(load16_guarded<E>(w + c, wend, left), load16_guarded<E>(x + c, xend, left), acc);
        }
    }
    return acc;
}

}  // namespace few
