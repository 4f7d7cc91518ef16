// direct_gemm.h -- the tiled product of tile_gemm.h for 16-bit and 8-bit operands whose rows are 16-byte aligned:
// memory goes to LDS without passing through registers (buffer loads to LDS), which leaves the registers to two sets
// of MFMA operands, so that the reads of one multiplication run under the one before.
//
// A step is 128 bytes of the contraction (64 or 128 values).  An operand lies in LDS as
//   DirectRows  [row][c], c along memory: 8 chunks of 16 bytes a row, in slots q ^ (row & 7) as in tile_gemm.h
//   DirectCols  [c][row], rows along memory (16-bit types): read transposed (ds_read_b64_tr_b16: 16 lanes give the
//               addresses of a 4 x 16 block, 8 bytes each, and get a row of 4 values each); blocks of 32 bytes are
//               exclusive-ored with c & 3, so that the four c of a block lie in different banks
// A load to LDS writes 16 bytes a lane in lane order, so it is the lane's source address that carries the permutation.
// Whatever lies behind the end of the operand (rows, the last values of c) reads as zero through the bounds of the
// buffer descriptor: there is no other code for the edges.
#pragma once

#include "tile_gemm.h"

namespace tile {

typedef __attribute__((address_space(3))) const char *lds_ptr;
__device__ __forceinline__ uint32_t lds_address(const void *p) { return (uint32_t)(uintptr_t)(lds_ptr)p; }

// a raw buffer of `bytes` (at most 2^31 - 1 count) from p
__device__ __forceinline__ u32x4 descriptor(const char *p, long long bytes)
{
    const uint64_t a = (uint64_t)p;
    const long long n = bytes < 0 ? 0 : bytes > 0x7FFFFFFF ? 0x7FFFFFFF : bytes;
    return u32x4{(uint32_t)a, (uint32_t)(a >> 32), (uint32_t)n, 0x00020000u};
}
// 16 bytes a lane to LDS at `to` + 16 lane.  No register is written; completion counts in vmcnt.
__device__ __forceinline__ void load_to_lds(u32x4 desc, uint32_t voffset, uint32_t soffset, uint32_t to)
{
    asm volatile("s_mov_b32 m0, %3\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, %2 offen lds" ::"v"(voffset), "s"(desc), "s"(soffset), "s"(to));
}
template <int N> __device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }

template <class T, int ROWS, int THREADS> struct DirectRows {
    static constexpr int N = ROWS * 8 / THREADS, ECH = T::ECH, STEP = 8 * ECH, READS = 1;   // instructions of read()
    const char *base;
    long long left;                          // bytes from base to the end of the tensor
    uint32_t voffset, hop, q;                // hop: bytes between this thread's rows
    int count;

    __device__ __forceinline__ void init(const typename T::elem *row0, long long ld, int, int c_count, const typename T::elem *end)
    {
        base = (const char *)row0;
        left = (const char *)end - base;
        count = c_count;
        const int r = threadIdx.x / 8;
        q = (threadIdx.x & 7) ^ (r & 7);
        voffset = (uint32_t)r * (uint32_t)(ld * sizeof(typename T::elem)) + q * 16;
        hop = (uint32_t)(THREADS / 8) * (uint32_t)(ld * sizeof(typename T::elem));
    }
    __device__ __forceinline__ void issue(int c0, uint32_t lds) const
    {
        const u32x4 d = descriptor(base + (long long)c0 * sizeof(typename T::elem), left - (long long)c0 * sizeof(typename T::elem));
        const uint32_t v = c0 + (int)q * ECH < count ? voffset : 0x80000000u;
        const uint32_t to = lds + __builtin_amdgcn_readfirstlane(threadIdx.x / 64) * 1024;
#pragma unroll
        for (int j = 0; j < N; ++j) load_to_lds(d, v, j * hop, to + j * THREADS * 16);
    }
    // the 16 rows from `row` (a multiple of 16), chunks 4 s .. 4 s + 3
    static __device__ __forceinline__ u32x4 read(const char *lds, int row, int s)
    {
        const int lane = threadIdx.x & 63;
        return *reinterpret_cast<const u32x4 *>(lds + lds_at<8>(lane & 15, 4 * s + (lane >> 4)) + row * 128);
    }
};

template <class T, int ROWS, int THREADS> struct DirectCols {
    static constexpr int SLOTS = ROWS / 8, N = 64 * SLOTS / THREADS, STEP = 64, READS = 2;
    static_assert(sizeof(typename T::elem) == 2 && THREADS / SLOTS % 4 == 0, "16-bit types");
    const char *base;
    long long ld, left;                      // bytes; left: from base to the end of the last c's part of this tile
    uint32_t voffset, hop;

    __device__ __forceinline__ void init(const typename T::elem *row0, long long ld_, int rows, int c_count, const typename T::elem *)
    {
        base = (const char *)row0;
        ld = ld_ * 2;
        left = (c_count - 1) * ld + rows * 2;
        const int c = threadIdx.x / SLOTS, slot = threadIdx.x % SLOTS;
        voffset = (uint32_t)c * (uint32_t)ld + ((((slot >> 1) ^ (c & 3)) << 1) | (slot & 1)) * 16;
        hop = (uint32_t)(THREADS / SLOTS) * (uint32_t)ld;
    }
    __device__ __forceinline__ void issue(int c0, uint32_t lds) const
    {
        const u32x4 d = descriptor(base + c0 * ld, left - c0 * ld);
        const uint32_t to = lds + __builtin_amdgcn_readfirstlane(threadIdx.x / 64) * 1024;
#pragma unroll
        for (int j = 0; j < N; ++j) load_to_lds(d, voffset, j * hop, to + j * THREADS * 16);
    }
    static __device__ __forceinline__ u32x4 read(const char *lds, int row, int s)
    {
        typedef short s4 __attribute__((ext_vector_type(4)));
        typedef __attribute__((address_space(3))) s4 *ptr;
        typedef uint32_t u2 __attribute__((ext_vector_type(2)));
        const int lane = threadIdx.x & 63, g = lane >> 4, j = lane & 15;
        const char *p = lds + (8 * g + (j >> 2)) * (ROWS * 2) + (j & 3) * 8 + (((row >> 4 & 3) ^ (j >> 2)) << 5) + (row >> 6) * 128 + s * (32 * ROWS * 2);
        const u2 a = __builtin_bit_cast(u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((ptr)(p)));
        const u2 b = __builtin_bit_cast(u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((ptr)(p + 4 * ROWS * 2)));
        return u32x4{a[0], a[1], b[0], b[1]};
    }
};

template <class S, class DA, class DB> struct DirectFragments {
    typedef typename S::T T;
    u32x4 a[S::NI], b[S::MI];
    __device__ __forceinline__ void read(const char *lds, int s)
    {
        const int wave = threadIdx.x >> 6;
#pragma unroll
        for (int n = 0; n < S::NI; ++n) a[n] = DA::read(lds, __builtin_amdgcn_readfirstlane(wave % S::WN * (S::BN / S::WN)) + 16 * n, s);
#pragma unroll
        for (int m = 0; m < S::MI; ++m) b[m] = DB::read(lds + S::A_BYTES, __builtin_amdgcn_readfirstlane(wave / S::WN * (S::BM / S::WM)) + 16 * m, s);
    }
    __device__ __forceinline__ void multiply(typename S::Acc &acc) const
    {
#pragma unroll
        for (int m = 0; m < S::MI; ++m)
#pragma unroll
            for (int n = 0; n < S::NI; ++n) acc[m][n] = T::mma(a[n], b[m], acc[m][n]);
    }
    // adds the values of B's rows over this lane's c
    __device__ __forceinline__ void add_up(float (&sum)[S::MI]) const
    {
#pragma unroll
        for (int m = 0; m < S::MI; ++m)
#pragma unroll
            for (int d = 0; d < 4; ++d)
                sum[m] += to_float(__builtin_bit_cast(typename T::elem, (uint16_t)b[m][d])) +
                          to_float(__builtin_bit_cast(typename T::elem, (uint16_t)(b[m][d] >> 16)));
    }
};

// As product() in tile_gemm.h: two steps in LDS, one barrier a step, before its second multiplication.  Behind it the
// loads of the next step have landed (they were issued a step ago) and nobody reads this one any more, so the loads of the
// step after the next may overwrite it.
template <class S, bool SUMS = false, class DA, class DB>
__device__ __forceinline__ void product_direct(const DA &a, const DB &b, int count, char *lds, typename S::Acc &acc, bool sums = false,
                                               float *sum = nullptr)
{
    constexpr int STEP = DA::STEP, HALF = S::A_BYTES + S::B_BYTES;
    static_assert(DA::STEP == DB::STEP, "one step for both operands");
    constexpr int MFMA = S::NI * S::MI, READS = S::NI * DA::READS + S::MI * DB::READS;
    const uint32_t at = lds_address(lds);
    DirectFragments<S, DA, DB> f[2];
    float add[S::MI] = {};
    a.issue(0, at);
    b.issue(0, at + S::A_BYTES);
    if (count > STEP) {
        a.issue(STEP, at + HALF);
        b.issue(STEP, at + HALF + S::A_BYTES);
        wait_loads<DA::N + DB::N>();
    } else {
        wait_loads<0>();
    }
    __syncthreads();
    f[0].read(lds, 0);
    int here = 0;
    for (int c0 = 0; c0 < count; c0 += STEP) {
        f[1].read(lds + here, 1);
        f[0].multiply(acc);
        interleave<MFMA, READS, 0, 0>();
        if constexpr (SUMS)
            if (sums) f[0].add_up(add);
        wait_loads<0>();
        __syncthreads();
        if (c0 + 2 * STEP < count) {
            a.issue(c0 + 2 * STEP, at + here);
            b.issue(c0 + 2 * STEP, at + here + S::A_BYTES);
        }
        here = HALF - here;
        f[0].read(lds + here, 0);
        f[1].multiply(acc);
        interleave<MFMA, READS, 0, 0>();
        if constexpr (SUMS)
            if (sums) f[1].add_up(add);
    }
    __syncthreads();
    if constexpr (SUMS) {
        if (sums) {                          // lanes i, i + 16, i + 32, i + 48 hold the row's four parts
#pragma unroll
            for (int m = 0; m < S::MI; ++m) {
                float v = add[m];
                v += __shfl_xor(v, 16, 64);
                v += __shfl_xor(v, 32, 64);
                sum[m] = v;
            }
        }
    }
}

inline bool direct_ok(const void *p, long long ld_bytes) { return ((uintptr_t)p & 15) == 0 && ld_bytes % 16 == 0; }

}  // namespace tile
