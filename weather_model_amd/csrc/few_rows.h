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

// This wave's share of the products of matrix row w (i = lane & 15: four consecutive rows of the result per lane) with a row of x;
// rows that do not exist are given as any that do.  x(c, left) gives the piece of the row from value c on, of which `left` count.
// begin() may be called long before multiply(): the first loads of the weights are then under way.
template <class T> struct Dot {
    typedef typename T::elem E;
    static constexpr int ROUND = 128 / sizeof(E), PIECE = 16 / sizeof(E);
    const E *w, *end;
    int K, rounds;
    u32x4 a[UNROLL][2];
    static __device__ __forceinline__ int at() { return (int)((threadIdx.x & 63) >> 4) * 2 * PIECE; }      // of this lane in a round
    __device__ __forceinline__ void load(int r)
    {
#pragma unroll
        for (int u = 0; u < UNROLL; ++u)
#pragma unroll
            for (int h = 0; h < 2; ++h) a[u][h] = *reinterpret_cast<const u32x4u *>(w + (r + u * WAVES) * ROUND + h * PIECE);
    }
    __device__ __forceinline__ bool batch(int r) const { return r + (UNROLL - 1) * WAVES < rounds; }
    __device__ __forceinline__ void begin(const E *row, const E *tensor_end, int K_)
    {
        w = row + at();
        end = tensor_end;
        K = K_;
        rounds = K / ROUND;
        if (batch(threadIdx.x >> 6)) load(threadIdx.x >> 6);
    }
    template <class X> __device__ __forceinline__ typename T::acc multiply(X x)
    {
        typename T::acc acc = {0, 0, 0, 0};
        int r = threadIdx.x >> 6;
        for (bool there = true; batch(r); r += UNROLL * WAVES, there = false) {
            u32x4 b[UNROLL][2];
            if (!there) load(r);
#pragma unroll
            for (int u = 0; u < UNROLL; ++u)
#pragma unroll
                for (int h = 0; h < 2; ++h) b[u][h] = x((r + u * WAVES) * ROUND + h * PIECE + at(), PIECE);
#pragma unroll
            for (int u = 0; u < UNROLL; ++u)
#pragma unroll
                for (int h = 0; h < 2; ++h) acc = piece<T>(a[u][h], b[u][h], acc);
        }
        for (; r * ROUND < K; r += WAVES)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int c = r * ROUND + h * PIECE, left = K - c - at();
                acc = piece<T>(load16_guarded<E>(w + c, end, left), x(c + at(), left), acc);
            }
        return acc;
    }
};
// x as a row in memory
template <class T> struct RowOf {
    const typename T::elem *x, *end;
    __device__ __forceinline__ u32x4 operator()(int c, int left) const
    {
        if (left >= (int)(16 / sizeof(typename T::elem))) return *reinterpret_cast<const u32x4u *>(x + c);
        return load16_guarded<typename T::elem>(x + c, end, left);
    }
};

}  // namespace few
