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
// rows that do not exist are given as any that do.  x gives the pieces of its row: whole(c) from value c on, part(c, left) of which
// only `left` values count.
// UNROLL: rounds whose loads go out together.  WAVES: of the workgroup.  EARLY: begin() is called long before multiply(), and the first loads of the weights
// go out there.
template <class T, int UNROLL, int WAVES, bool EARLY = false> struct Dot {
    typedef typename T::elem E;
    static constexpr int ROUND = 128 / sizeof(E), PIECE = 16 / sizeof(E);
    typedef u32x4 Batch[UNROLL][2];
    const E *w, *end;
    int K, rounds;                           // rounds: whole ones
    Batch first;
    static __device__ __forceinline__ int wave() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }
    static __device__ __forceinline__ int at() { return (int)((threadIdx.x & 63) >> 4) * 2 * PIECE; }      // of this lane in a round
    // UNROLL rounds from r on, WAVES apart; behind the last whole one that one again
    __device__ __forceinline__ int round(int r, int u) const { return min(r + u * WAVES, rounds - 1) * ROUND; }
    __device__ __forceinline__ void load(int r, Batch &to) const
    {
#pragma unroll
        for (int u = 0; u < UNROLL; ++u)
#pragma unroll
            for (int h = 0; h < 2; ++h) to[u][h] = *reinterpret_cast<const u32x4u *>(w + round(r, u) + h * PIECE);
    }
    template <class X> __device__ __forceinline__ void add(int r, const Batch &a, const X &x, typename T::acc &acc) const
    {
        Batch b;
#pragma unroll
        for (int u = 0; u < UNROLL; ++u)
#pragma unroll
            for (int h = 0; h < 2; ++h) b[u][h] = x.whole(round(r, u) + h * PIECE + at());
#pragma unroll
        for (int u = 0; u < UNROLL; ++u)
            if (r + u * WAVES < rounds)
#pragma unroll
                for (int h = 0; h < 2; ++h) acc = piece<T>(a[u][h], b[u][h], acc);
    }
    __device__ __forceinline__ void begin(const E *row, const E *tensor_end, int K_)
    {
        w = row + at();
        end = tensor_end;
        K = K_;
        rounds = K / ROUND;
        if constexpr (EARLY)
            if (wave() < rounds) load(wave(), first);
    }
    template <class X> __device__ __forceinline__ typename T::acc multiply(const X &x) const
    {
        typename T::acc acc = {0, 0, 0, 0};
        int r = wave();
        if constexpr (EARLY) {
            if (r < rounds) add(r, first, x, acc);
            r += UNROLL * WAVES;
        }
        for (; r < rounds; r += UNROLL * WAVES) {
            Batch a;
            load(r, a);
            add(r, a, x, acc);
        }
        if (rounds * ROUND < K && rounds % WAVES == wave())
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int c = rounds * ROUND + h * PIECE, left = K - c - at();
                acc = piece<T>(load16_of_row<E>(w - at(), c + at(), K, end), x.part(c + at(), left), acc);
            }
        return acc;
    }
};
// x as a row in memory
template <class T> struct RowOf {
    const typename T::elem *x, *end;
    __device__ __forceinline__ u32x4 whole(int c) const { return *reinterpret_cast<const u32x4u *>(x + c); }
    __device__ __forceinline__ u32x4 part(int c, int left) const { return load16_of_row<typename T::elem>(x, c, c + left, end); }
};

}  // namespace few
