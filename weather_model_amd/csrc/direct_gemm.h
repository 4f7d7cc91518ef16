// direct_gemm.h -- the tiled product of tile_gemm.h for 16-bit and 8-bit operands whose rows are 16-byte aligned:
// memory goes to LDS without passing through registers (buffer loads to LDS), which leaves the registers to two sets
// of MFMA operands, so that the reads of one multiplication run under the one before.
//
// Bound by the matrix unit: 16384 rows, 16 experts of 2048 -> 4096 bf16, evenly spread, 266 us = 1030 TFLOP/s, where a library product of
// 8192^3 makes 1360; a stage in the loop runs at 1430.  What is lost is the ring's fill and the way out of each tile (5 and 6 us of
// 27 a round) and, with uneven experts (300 us), their last rows.
//
// A stage is 64 bytes of the contraction (32 or 64 values), one MFMA deep; LDS holds a ring of them (256 x 256: of 5, 160 KB; of 4
// 308 us instead of 299).  An operand lies as
//   DirectRows  [row][c], c along memory: 4 chunks of 16 bytes a row, two rows a line, placed by lds_at<4> of tile_gemm.h
//   DirectCols  [c][row], rows along memory (16-bit types): read transposed (ds_read_b64_tr_b16: 16 lanes give the
//               addresses of a 4 x 16 block, 8 bytes each, and get a row of 4 values each); blocks of 32 bytes are
//               exclusive-ored with bits of c, so that what is read together lies in different banks
// A load to LDS writes 16 bytes a lane in lane order, so it is the lane's source address that carries the permutation.
// Whatever lies behind the end of the operand (rows, the last values of c) reads as zero through the bounds of the
// buffer descriptor: there is no other code for the edges.
#pragma once

#include "tile_gemm.h"

namespace tile {

typedef __attribute__((address_space(3))) const char *lds_ptr;
__device__ __forceinline__ uint32_t lds_address(const void *p) { return (uint32_t)(uintptr_t)(lds_ptr)p; }

// a raw buffer of `bytes` (at most 2^31 - 1 count) from p.  A word whose voffset + soffset lies beyond them reads as zero, also where
// soffset alone does; the sum does not wrap.
__device__ __forceinline__ u32x4 descriptor(const char *p, long long bytes)
{
    const uint64_t a = (uint64_t)p;
    const long long n = bytes < 0 ? 0 : bytes > 0x7FFFFFFF ? 0x7FFFFFFF : bytes;
    return u32x4{(uint32_t)a, (uint32_t)(a >> 32), (uint32_t)n, 0x00020000u};
}
// 16 bytes a lane to LDS at `to` + 16 lane.  No register is written; completion counts in vmcnt.
__device__ __forceinline__ void load_to_lds(u32x4 desc, uint32_t voffset, uint32_t soffset, uint32_t to)
{
    asm volatile("s_mov_b32 m0, %3\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, %2 offen lds" ::"v"(voffset), "s"(desc), "s"(soffset), "s"(to) : "m0");
}
template <int N> __device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }

// The stages are issued in order: issue() moves on by one.
template <class T, int ROWS, int THREADS> struct DirectRows {
    static constexpr int BYTES = ROWS * 64, N = BYTES / (THREADS * 16), ECH = T::ECH, STEP = 4 * ECH, READS = 1;   // READS: instructions of read()
    u32x4 desc;
    uint32_t voffset, hop, soffset;          // hop: bytes between this thread's rows
    int left;                                // values of c from this lane's chunk on

    __device__ __forceinline__ void init(const typename T::elem *row0, long long ld, int, int c_count, const typename T::elem *end)
    {
        desc = descriptor((const char *)row0, (const char *)end - (const char *)row0);
        // lane order in LDS: lines of 128 bytes, each two rows of four chunks
        const int line = threadIdx.x / 8, h = (line & 3) | (((line ^ (line >> 1)) & 1) << 2), at = (threadIdx.x & 7) ^ h;
        const int r = line * 2 + (at >> 2), q = at & 3;
        voffset = (uint32_t)r * (uint32_t)(ld * sizeof(typename T::elem)) + q * 16;
        hop = (uint32_t)(THREADS / 4) * (uint32_t)(ld * sizeof(typename T::elem));
        soffset = 0;
        left = c_count - q * ECH;
    }
    __device__ __forceinline__ void issue(uint32_t lds)
    {
        const uint32_t v = left > 0 ? voffset : 0x80000000u;
        const uint32_t to = lds + __builtin_amdgcn_readfirstlane(threadIdx.x / 64) * 1024;
#pragma unroll
        for (int j = 0; j < N; ++j) load_to_lds(desc, v, soffset + j * hop, to + j * THREADS * 16);
        soffset += 64;
        left -= STEP;
    }
    // the 16 rows from `row` (a multiple of 16)
    static __device__ __forceinline__ u32x4 read(const char *lds, int row)
    {
        const int lane = threadIdx.x & 63;
        return *reinterpret_cast<const u32x4 *>(lds + lds_at<4>(lane & 15, lane >> 4) + row * 64);
    }
};

template <class T, int ROWS, int THREADS> struct DirectCols {
    static constexpr int BYTES = ROWS * 64, SLOTS = ROWS / 8, N = BYTES / (THREADS * 16), STEP = 32, READS = 2, HOP = THREADS / SLOTS,
                         SHARE = STEP * ROWS / 2 / THREADS;
    static_assert(sizeof(typename T::elem) == 2 && HOP % 8 == 0, "16-bit types");
    const char *at;
    long long ld, left;                      // bytes; left: from `at` to the end of the last c's part of this tile
    uint32_t voffset[2];                     // of this thread's even and odd hops
    // the permutation of 32-byte blocks at c (bits 2 and 5 are fixed in a read instruction)
    static __device__ __forceinline__ int mix(int c) { return ((c & 3) | ((((c >> 3) ^ (c >> 4)) & 1) << 2)) & (ROWS / 16 - 1); }

    __device__ __forceinline__ void init(const typename T::elem *row0, long long ld_, int rows, int c_count, const typename T::elem *)
    {
        at = (const char *)row0;
        ld = ld_ * 2;
        left = (c_count - 1) * ld + rows * 2;
        const int c = threadIdx.x / SLOTS, slot = threadIdx.x % SLOTS;
#pragma unroll
        for (int k = 0; k < 2; ++k)
            voffset[k] = (uint32_t)c * (uint32_t)ld + ((((slot >> 1) ^ mix(c + k * HOP)) << 1) | (slot & 1)) * 16;
    }
    __device__ __forceinline__ void issue(uint32_t lds)
    {
        const u32x4 d = descriptor(at, left);
        const uint32_t to = lds + __builtin_amdgcn_readfirstlane(threadIdx.x / 64) * 1024;
#pragma unroll
        for (int j = 0; j < N; ++j) load_to_lds(d, voffset[j & 1], j * HOP * (uint32_t)ld, to + j * THREADS * 16);
        at += STEP * ld;
        left -= STEP * ld;
    }
    // Sums over c of two rows of the tile, threadIdx.x % (ROWS / 2) * 2 and the next, over the SHARE c that fall to this thread:
    // the sums of a stage are spread evenly over all threads, as one thread that is late holds up the barrier for all.
    static __device__ __forceinline__ void add_up(const char *lds, float (&sum)[2])
    {
        const int pair = threadIdx.x % (ROWS / 2), c0 = threadIdx.x / (ROWS / 2) * SHARE;
        uint32_t v[SHARE];
#pragma unroll
        for (int e = 0; e < SHARE; ++e)
            v[e] = *reinterpret_cast<const uint32_t *>(lds + (c0 + e) * (ROWS * 2) + ((pair / 8 ^ mix(c0 + e)) << 5) + pair % 8 * 4);
#pragma unroll
        for (int e = 0; e < SHARE; ++e) {
            sum[0] += to_float(__builtin_bit_cast(typename T::elem, (uint16_t)v[e]));
            sum[1] += to_float(__builtin_bit_cast(typename T::elem, (uint16_t)(v[e] >> 16)));
        }
    }
    // their total, of row threadIdx.x < ROWS, in a fixed order; LDS holds 32 / SHARE x ROWS floats
    static __device__ __forceinline__ float total(float *lds, const float (&sum)[2])
    {
        const int pair = threadIdx.x % (ROWS / 2);
        float *own = lds + threadIdx.x / (ROWS / 2) * ROWS + 2 * pair;
        own[0] = sum[0];
        own[1] = sum[1];
        __syncthreads();
        float s = 0.0f;
        if (threadIdx.x < ROWS)
#pragma unroll
            for (int k = 0; k < STEP / SHARE; ++k) s += lds[k * ROWS + threadIdx.x];
        return s;
    }
    static __device__ __forceinline__ u32x4 read(const char *lds, int row)
    {
        typedef short s4 __attribute__((ext_vector_type(4)));
        typedef __attribute__((address_space(3))) s4 *ptr;
        typedef uint32_t u2 __attribute__((ext_vector_type(2)));
        const int lane = threadIdx.x & 63, c = 8 * (lane >> 4) + ((lane & 15) >> 2);
        const char *p = lds + c * (ROWS * 2) + (lane & 3) * 8 + (((row >> 4 & 7) ^ mix(c)) << 5) + (row >> 7) * 256;
        const u2 a = __builtin_bit_cast(u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((ptr)(p)));
        const u2 b = __builtin_bit_cast(u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((ptr)(p + 4 * ROWS * 2)));
        return u32x4{a[0], a[1], b[0], b[1]};
    }
};

template <class S, class DA, class DB> struct DirectFragments {
    typedef typename S::T T;
    u32x4 a[S::NI], b[S::MI];
    __device__ __forceinline__ void read(const char *lds)
    {
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#pragma unroll
        for (int n = 0; n < S::NI; ++n) a[n] = DA::read(lds, wave % S::WN * (S::BN / S::WN) + 16 * n);
#pragma unroll
        for (int m = 0; m < S::MI; ++m) b[m] = DB::read(lds + DA::BYTES, wave / S::WN * (S::BM / S::WM) + 16 * m);
    }
    __device__ __forceinline__ void multiply(typename S::Acc &acc) const
    {
#pragma unroll
        for (int m = 0; m < S::MI; ++m)
#pragma unroll
            for (int n = 0; n < S::NI; ++n) acc[m][n] = T::mma(a[n], b[m], acc[m][n]);
    }
};

// Stage s is multiplied from registers while the operands of stage s + 1 are read.  The one barrier a stage lies before
// that: behind it stage s + 1 has landed (issued RING - 1 stages ago) and every wave has read stage s, so its place in the
// ring takes stage s + RING.  The loads behind the last stage are issued all the same, to a place that nobody reads
// and with nothing in their bounds, so that the count of loads in flight is always the same.
// A wave whose rows (of B, `rows` exist) all lie behind the end only takes part in the loads.
// SUMS: B's rows (DirectCols) are summed over c as well, into this thread's `sum`.
template <class S, int RING, bool SUMS, class DA, class DB>
__device__ __forceinline__ void product_direct(DA &a, DB &b, int count, int rows, char *lds, typename S::Acc &acc, float (&sum)[2])
{
    constexpr int STEP = DA::STEP, STAGE = DA::BYTES + DB::BYTES;
    static_assert(DA::STEP == DB::STEP, "one step for both operands");
    constexpr int MFMA = S::NI * S::MI, READS = S::NI * DA::READS + S::MI * DB::READS;
    const uint32_t base = lds_address(lds);
    DirectFragments<S, DA, DB> f[2];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#pragma unroll
    for (int k = 0; k < RING; ++k) {
        a.issue(base + k * STAGE);
        b.issue(base + k * STAGE + DA::BYTES);
    }
    wait_loads<(RING - 1) * (DA::N + DB::N)>();
    __syncthreads();
    int here = 0;                            // where the stage lies that is in registers
    auto next = [&]() {
        wait_loads<(RING - 2) * (DA::N + DB::N)>();
        __syncthreads();
        a.issue(base + here);
        b.issue(base + here + DA::BYTES);
        here = here == (RING - 1) * STAGE ? 0 : here + STAGE;
    };
    if (SUMS || wave / S::WN * (S::BM / S::WM) < rows) {
        f[0].read(lds);
        if constexpr (SUMS) DB::add_up(lds + DA::BYTES, sum);
        for (int c0 = 0; c0 < count; c0 += 2 * STEP) {
#pragma unroll
            for (int k = 0; k < 2; ++k) {    // an odd number of stages ends with one of zeros
                next();
                f[k ^ 1].read(lds + here);
                f[k].multiply(acc);
                interleave<MFMA, READS, 0, 0>();
                if constexpr (SUMS) DB::add_up(lds + here + DA::BYTES, sum);
            }
        }
    } else {
        for (int c0 = 0; c0 < count; c0 += 2 * STEP) {
            next();
            next();
        }
    }
    wait_loads<0>();
    __syncthreads();
}
template <class S, int RING, class DA, class DB>
__device__ __forceinline__ void product_direct(DA &a, DB &b, int count, int rows, char *lds, typename S::Acc &acc)
{
    float none[2];
    product_direct<S, RING, false>(a, b, count, rows, lds, acc, none);
}

// Whether tiles of 256 x 256, one a CU, end before those of 128 x 128, two a CU: by the rounds that each makes, the last of them cut (Cut).
// A round of the larger takes 1.5 times as long (1024 deep in bf16: 34 | 22 us); parts of a round as measured.  bf16, us, 128 | 256:
// 8 experts, 16384 rows of 1024 -> 1024 45 | 37, 12 experts, 20000 rows of 1000 -> 1000 81 | 63, 22 experts, 14612 rows of 2976 -> 1320
// 215 | 207 and backward 211 | 169, 2 experts, 30000 rows of 512 -> 640 33 | 36; 512 rows of 8192 -> 2048 37 | 59.
inline bool tiles_of_256(int G, int M, int N, int cus)
{
    if (M / G < 256 || N < 256) return false;
    const auto time = [&](int size, long long slots, int whole, int half, int quarter) {
        const long long t = ((long long)M / size + G / 2) * ((N + size - 1) / size), left = t % slots;
        return t / slots * whole + (left == 0 ? 0 : left * 4 <= slots ? quarter : left * 2 <= slots ? half : whole);
    };
    return time(256, cus, 100, 60, 38) < time(128, 2ll * cus, 68, 44, 36);
}

inline bool direct_ok(const void *p, long long ld_bytes) { return ((uintptr_t)p & 15) == 0 && ld_bytes % 16 == 0; }

}  // namespace tile
