// tile_gemm.h -- the tiled matrix product under the grouped Dense layers (grouped.hip) and the 8-bit
// integer product (int8.hip): operand loaders, the LDS layout, the MFMA core and the map from a
// workgroup to its tile of a ragged batch.
//
// A tile is C[i][j] = sum_c A[i][c] B[j][c], BN values of i (the output's contiguous side) by BM of j (its
// rows).  D of an MFMA has four consecutive i of one j in a lane, which makes a store one vector.
// LDS holds both operands as [row][c], `BKC` chunks of 16 bytes a row, whatever their layout in memory:
//   contiguous  c runs along memory: a chunk is one 16-byte load (two for float32)
//   strided     i (or j) runs along memory: a thread loads 8 c of a few rows and transposes in registers
//
// float32 is split into three bf16 pieces, 2^16 x = h + m + l (each the nearest to what is left: 24 bits), and a
// product is the six piece products that are not below 2^-24 of it: hh, hm, mh, hl, lh, mm, each exact in the
// float32 accumulator.  That is float32 accuracy (what is left out is 3 2^-26 of |a||b| at most) at 2500 / 6
// TFLOP/s of matrix rate where the float32 MFMA has 157.  The last bit of a subnormal x is 2^-149 and the last of bf16
// 2^-133, hence the factor: without it the third piece of |x| < 2^-109 lost bits (5e-5 of 2^-120, all of 2^-133).  It costs
// two multiplications a pair of values and the sums one by 2^-32 (8191 rows, 8 experts of 1024 -> 1024, forward and gradients
// 326 | 335 us, 45001 rows of 432 -> 216 72.8 | 74.5).  An infinity, a NaN or a value that rounds up to infinity in bf16
// (from 2^112 on) makes a NaN of its products, and a sum from 2^96 on may overflow in its first piece; elements of C that
// are not finite are summed again in float32 (not_finite_again).
#pragma once

#include <type_traits>

#include "half_types.h"

namespace tile {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32u __attribute__((aligned(1)));
typedef uint32_t u32x4u __attribute__((ext_vector_type(4), aligned(1)));
typedef bf16_t bf16x8 __attribute__((ext_vector_type(8)));
typedef f16_t f16x8 __attribute__((ext_vector_type(8)));
typedef f32x4 f32x4b __attribute__((aligned(16)));

// ---- element types
struct BF16 {
    typedef bf16_t elem;
    typedef f32x4 acc;
    static constexpr int PLANES = 1, BKC = 8, ECH = 8;      // pieces, chunks a row, elements a chunk
    static __device__ __forceinline__ acc mma(u32x4 a, u32x4 b, acc c)
    {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
};
struct F16 {
    typedef f16_t elem;
    typedef f32x4 acc;
    static constexpr int PLANES = 1, BKC = 8, ECH = 8;
    static __device__ __forceinline__ acc mma(u32x4 a, u32x4 b, acc c)
    {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
};
struct F32 {
    typedef float elem;
    typedef f32x4 acc;
    static constexpr int PLANES = 3, BKC = 4, ECH = 8;
    static __device__ __forceinline__ acc mma(u32x4 a, u32x4 b, acc c) { return BF16::mma(a, b, c); }
};
struct I8 {
    typedef int8_t elem;
    typedef i32x4 acc;
    static constexpr int PLANES = 1, BKC = 8, ECH = 16;
    static __device__ __forceinline__ acc mma(u32x4 a, u32x4 b, acc c)
    {
        return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, a), __builtin_bit_cast(i32x4, b), c, 0, 0, 0);
    }
};

// max(v, 0) that keeps a NaN
__device__ __forceinline__ float relu_of(float v) { return v < 0.0f ? 0.0f : v; }

// Byte address of chunk q of a row.  A line of 128 bytes is one row of eight chunks or two of four; the slot of a chunk
// in its line is exclusive-ored with the row, so that the 8 rows that a step of an MFMA operand's read touches, and the
// chunks that a step of a loader's write brings, lie in different banks.  16 rows on, the slots are the same again:
// an operand's other rows are immediate offsets.
template <int BKC> __device__ __forceinline__ int lds_at(int row, int q)
{
    if constexpr (BKC == 8) return row * 128 + ((q ^ (row & 7)) << 4);
    const int p = row >> 1, h = (p & 3) | (((p ^ (p >> 1)) & 1) << 2);
    return p * 128 + (((((row & 1) << 2) | q) ^ h) << 4);
}

// ---- global loads
// 16 bytes at p of which `avail` elements count; the rest read as zero.  Nothing at or beyond `end` is read.
template <class E> __device__ __forceinline__ u32x4 load16_guarded(const E *p, const E *end, int avail)
{
    constexpr int N = 16 / sizeof(E);
    u32x4 v = {0u, 0u, 0u, 0u};
    if (avail <= 0) return v;
    if (end - p >= N) {
        v = *reinterpret_cast<const u32x4u *>(p);
        if (avail < N) {
            const int bytes = avail * (int)sizeof(E);
#pragma unroll
            for (int d = 0; d < 4; ++d) {
                const int keep = bytes - 4 * d;
                v[d] = keep >= 4 ? v[d] : keep <= 0 ? 0u : v[d] & ((1u << (8 * keep)) - 1u);
            }
        }
        return v;
    }
    // one value after the other: the last bytes of a tensor, and no registers for it
    constexpr int PER_WORD = 4 / sizeof(E);
#pragma unroll
    for (int d = 0; d < 4; ++d)
#pragma unroll 1
        for (int i = 0; i < PER_WORD; ++i) {
            const int e = d * PER_WORD + i;
            if (e >= avail || p + e >= end) break;
            uint32_t bits;
            if constexpr (sizeof(E) == 4) bits = __builtin_bit_cast(uint32_t, p[e]);
            else if constexpr (sizeof(E) == 2) bits = __builtin_bit_cast(uint16_t, p[e]);
            else bits = (uint8_t)p[e];
            v[d] |= bits << (8 * (int)sizeof(E) * i);
        }
    return v;
}

// 16 bytes from value `pos` on of a row of `count` values that lie within a tensor ending at `end`; zeros behind the row.  Whatever would
// leave the row is read as its last 16 bytes and moved down: value after value, the one tile that meets the end of a tensor held up
// the launch (33 experts, 2999 rows, float16: 333 -> 515 forward 13.9 -> 11.4 us, gradients of rows 19.9 -> 17.9, of weights 25.4 -> 19.7).
template <class E> __device__ __forceinline__ u32x4 load16_of_row(const E *row, int pos, int count, const E *end)
{
    constexpr int N = 16 / sizeof(E);
    if (count < N) return load16_guarded<E>(row + pos, end, count - pos);
    const int at = min(pos, count - N), down = min((pos - at) * (int)sizeof(E), 16) * 8;
    const u32x4 v = *reinterpret_cast<const u32x4u *>(row + at);
    const uint64_t lo = (uint64_t)v[1] << 32 | v[0], hi = (uint64_t)v[3] << 32 | v[2];
    const uint64_t a = down == 0 ? lo : down < 64 ? lo >> down | hi << (64 - down) : down < 128 ? hi >> (down - 64) : 0,
                   b = down < 64 ? hi >> down : 0;
    return u32x4{(uint32_t)a, (uint32_t)(a >> 32), (uint32_t)b, (uint32_t)(b >> 32)};
}

__device__ __forceinline__ uint32_t pack_bf16(float a, float b)
{
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    typedef bf16_t b2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){a, b}, b2));
}
// the three pieces of a pair of float32 values times SPLIT_SCALE, packed; a sum of products is then to be multiplied by SPLIT_UNSCALE
constexpr float SPLIT_SCALE = 0x1p16f, SPLIT_UNSCALE = 0x1p-32f;
__device__ __forceinline__ void split2(float a, float b, uint32_t out[3])
{
    a *= SPLIT_SCALE;
    b *= SPLIT_SCALE;
#pragma unroll
    for (int p = 0; p < 3; ++p) {
        out[p] = pack_bf16(a, b);
        if (p < 2) {
            a -= __builtin_bit_cast(float, out[p] << 16);
            b -= __builtin_bit_cast(float, out[p] & 0xFFFF0000u);
        }
    }
}

// ---- operands.  load() brings a step of STEP values of c into registers without looking at the end of c; what lies behind the
// end is made zero by trim() before store().  That reads up to STEP - 1 values too many, which `safe` says lie within the
// tensor; where they do not, the last step takes load_guarded(), which reads nothing beyond what it is to read.

// c along memory: rows of `ld` elements, ROWS of them a tile
template <class T, int ROWS, int THREADS> struct Contiguous {
    typedef typename T::elem E;
    static constexpr int BKC = T::BKC, STEP = BKC * T::ECH, PER = ROWS * BKC / THREADS, LOADS = T::PLANES == 3 ? 2 : 1;
    static constexpr int N_LOADS = PER * LOADS, N_STORES = PER * T::PLANES;      // instructions of load() and store()
    static_assert(PER >= 1, "tile too small for the workgroup");
    struct Regs {
        u32x4 v[PER][LOADS];
    };
    const E *base, *end;                     // (row 0 of the tile, c = 0) and the end of the tensor
    uint32_t off[PER];                       // element offset of this thread's rows, chunk included
    int q, count;                            // count: values of c there are
    bool safe;
    static constexpr bool slow = false;      // every whole step can take load()

    // rows_left >= 1: rows from row0 on that exist; later ones repeat the last
    __device__ __forceinline__ void init(const E *tensor_row0, long long ld, int rows_left, int c_count, const E *tensor_end)
    {
        base = tensor_row0;
        end = tensor_end;
        count = c_count;
        q = threadIdx.x % BKC;
        safe = end - base >= (long long)(min(ROWS, rows_left) - 1) * ld + (c_count + STEP - 1) / STEP * STEP;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const int r = threadIdx.x / BKC + j * (THREADS / BKC);
            off[j] = (uint32_t)((long long)min(r, rows_left - 1) * ld) + (uint32_t)(q * T::ECH);
        }
    }
    __device__ __forceinline__ void load(Regs &reg, int c0) const
    {
        const E *at = base + c0;
#pragma unroll
        for (int j = 0; j < PER; ++j)
#pragma unroll
            for (int h = 0; h < LOADS; ++h) reg.v[j][h] = *reinterpret_cast<const u32x4u *>(at + off[j] + h * 4);
    }
    __device__ __forceinline__ void trim(Regs &reg, int c0) const
    {
#pragma unroll
        for (int h = 0; h < LOADS; ++h) {
            const int bytes = (count - c0 - q * T::ECH) * (int)sizeof(E) - h * 16;
#pragma unroll
            for (int d = 0; d < 4; ++d) {
                const int keep = bytes - 4 * d;
                const uint32_t m = keep >= 4 ? 0xFFFFFFFFu : keep <= 0 ? 0u : (1u << (8 * keep)) - 1u;
#pragma unroll
                for (int j = 0; j < PER; ++j) reg.v[j][h][d] &= m;
            }
        }
    }
    __device__ __forceinline__ void load_guarded(Regs &reg, int c0) const
    {
        const int pos = c0 + q * T::ECH;
#pragma unroll
        for (int j = 0; j < PER; ++j)
#pragma unroll
            for (int h = 0; h < LOADS; ++h) reg.v[j][h] = load16_of_row<E>(base + off[j] - q * T::ECH, pos + h * 4, count, end);
    }
    __device__ __forceinline__ void store(const Regs &reg, char *lds) const
    {
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const int r = threadIdx.x / BKC + j * (THREADS / BKC);
            if constexpr (T::PLANES == 1) {
                *reinterpret_cast<u32x4 *>(lds + lds_at<BKC>(r, q)) = reg.v[j][0];
            } else {
                u32x4 piece[3];
#pragma unroll
                for (int d = 0; d < 4; ++d) {
                    uint32_t o[3];
                    const f32x4 f = __builtin_bit_cast(f32x4, reg.v[j][d / 2]);
                    split2(f[2 * (d & 1)], f[2 * (d & 1) + 1], o);
#pragma unroll
                    for (int p = 0; p < 3; ++p) piece[p][d] = o[p];
                }
#pragma unroll
                for (int p = 0; p < 3; ++p)
                    *reinterpret_cast<u32x4 *>(lds + p * (ROWS * BKC * 16) + lds_at<BKC>(r, q)) = piece[p];
            }
        }
    }
};

// the tile's rows along memory: element (row r, c) at base + c * ld + r; THREADS of the workgroup load it, from number `first` on
template <class T, int ROWS, int THREADS> struct Strided {
    typedef typename T::elem E;
    static constexpr int BKC = T::BKC, STEP = BKC * 8, BLOCKS = THREADS / BKC, W = ROWS / BLOCKS;   // W rows x 8 c a thread
    static constexpr int WORDS = W * sizeof(E) / 4, PER_WORD = 4 / sizeof(E);
    static constexpr int N_LOADS = 8, N_STORES = W * T::PLANES;
    static_assert(WORDS >= 1 && T::ECH == 8, "tile too small for the workgroup");
    typedef uint32_t words __attribute__((ext_vector_type(WORDS), aligned(sizeof(E))));
    struct Regs {
        uint32_t v[8][WORDS];
    };
    const E *base;
    long long ld;
    int r0, q, count;
    float sum[W];                            // of what add_up() saw
    int most;                                // rows that exist, at least 1
    bool safe;
    bool slow;                               // fewer rows than a thread's vector: load() does not fit (workgroup-uniform)

    __device__ __forceinline__ void init(const E *tensor_row0, long long ld_, int rows_left, int c_count, const E *end, int first = 0)
    {
        base = tensor_row0;
        ld = ld_;
        count = c_count;
        q = threadIdx.x % BKC;
        most = rows_left;
        slow = rows_left < W;
        safe = end - base >= ((c_count + STEP - 1) / STEP * STEP - 1) * ld + min(ROWS, rows_left);
#pragma unroll
        for (int i = 0; i < W; ++i) sum[i] = 0.0f;
        // a vector that would leave the rows moves back into them: two threads then write the same values to the
        // same place, and rows that do not exist keep whatever LDS held (their results are not stored)
        r0 = slow ? 0 : min(((int)threadIdx.x - first) / BKC * W, rows_left - W);
    }
    __device__ __forceinline__ void load(Regs &reg, int c0) const
    {
        const E *at = base + (long long)c0 * ld;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const E *p = at + e * ld + (uint32_t)(q * 8 * (int)ld + r0);       // scalar base, one offset register
            if constexpr (WORDS == 1) {
                reg.v[e][0] = *reinterpret_cast<const u32u *>(p);
            } else {
                const words v = *reinterpret_cast<const words *>(p);
#pragma unroll
                for (int w = 0; w < WORDS; ++w) reg.v[e][w] = v[w];
            }
        }
    }
    __device__ __forceinline__ void trim(Regs &reg, int c0) const
    {
#pragma unroll
        for (int e = 0; e < 8; ++e)
#pragma unroll
            for (int w = 0; w < WORDS; ++w) reg.v[e][w] = c0 + q * 8 + e < count ? reg.v[e][w] : 0u;
    }
    __device__ __forceinline__ void load_guarded(Regs &reg, int c0) const
    {
        // the last c again for those behind it, and the last row
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const E *p = base + (long long)min(c0 + q * 8 + e, count - 1) * ld;
            if (slow) {
#pragma unroll
                for (int w = 0; w < WORDS; ++w)
                    if constexpr (PER_WORD == 1) reg.v[e][w] = __builtin_bit_cast(uint32_t, p[min(r0 + w, most - 1)]);
                    else
                        reg.v[e][w] = (uint32_t)__builtin_bit_cast(uint16_t, p[min(r0 + 2 * w, most - 1)]) |
                                      (uint32_t)__builtin_bit_cast(uint16_t, p[min(r0 + 2 * w + 1, most - 1)]) << 16;
            } else if constexpr (WORDS == 1) {
                reg.v[e][0] = *reinterpret_cast<const u32u *>(p + r0);
            } else {
                const words v = *reinterpret_cast<const words *>(p + r0);
#pragma unroll
                for (int w = 0; w < WORDS; ++w) reg.v[e][w] = v[w];
            }
        }
        trim(reg, c0);
    }
    // adds what the registers hold to the sums of this thread's rows over c
    __device__ __forceinline__ void add_up(const Regs &reg)
    {
#pragma unroll
        for (int e = 0; e < 8; ++e)
#pragma unroll
            for (int i = 0; i < W; ++i) {
                if constexpr (sizeof(E) == 4) sum[i] += __builtin_bit_cast(float, reg.v[e][i]);
                else sum[i] += to_float(__builtin_bit_cast(E, (uint16_t)(reg.v[e][i / 2] >> (16 * (i & 1)))));
            }
    }
    // the sums over all c, in a fixed order: LDS holds BKC x ROWS floats; returns that of row threadIdx.x < ROWS
    __device__ __forceinline__ float total(float *lds, bool mine = true) const
    {
        if (mine)
#pragma unroll
            for (int i = 0; i < W; ++i) lds[q * ROWS + r0 + i] = sum[i];
        __syncthreads();
        float s = 0.0f;
        if (threadIdx.x < ROWS)
#pragma unroll
            for (int k = 0; k < BKC; ++k) s += lds[k * ROWS + threadIdx.x];
        return s;
    }
    __device__ __forceinline__ void store(const Regs &reg, char *lds) const
    {
#pragma unroll
        for (int i = 0; i < W; ++i) {
            const int r = r0 + i;
            if constexpr (T::PLANES == 1) {
                u32x4 v;
#pragma unroll
                for (int d = 0; d < 4; ++d)
                    v[d] = __builtin_amdgcn_perm(reg.v[2 * d + 1][i / 2], reg.v[2 * d][i / 2], i & 1 ? 0x07060302u : 0x05040100u);
                *reinterpret_cast<u32x4 *>(lds + lds_at<BKC>(r, q)) = v;
            } else {
                u32x4 piece[3];
#pragma unroll
                for (int d = 0; d < 4; ++d) {
                    uint32_t o[3];
                    split2(__builtin_bit_cast(float, reg.v[2 * d][i]), __builtin_bit_cast(float, reg.v[2 * d + 1][i]), o);
#pragma unroll
                    for (int p = 0; p < 3; ++p) piece[p][d] = o[p];
                }
#pragma unroll
                for (int p = 0; p < 3; ++p)
                    *reinterpret_cast<u32x4 *>(lds + p * (ROWS * BKC * 16) + lds_at<BKC>(r, q)) = piece[p];
            }
        }
    }
};

// Two strided operands of as many rows each: one half of the waves loads the one, the other half the other, so that a thread's
// loads are twice as wide.  Stands in both places of product().
template <class T, int ROWS, int THREADS> struct StridedPair : Strided<T, ROWS, THREADS / 2> {
    typedef Strided<T, ROWS, THREADS / 2> Half;
    typedef typename T::elem E;
    typedef typename Half::Regs Regs;
    bool second;
    __device__ __forceinline__ void init(const E *a, long long lda, int rows_a, const E *a_end, const E *b, long long ldb, int rows_b, const E *b_end,
                                         int count)
    {
        Half other;                          // the bounds of both halves hold for all waves
        second = __builtin_amdgcn_readfirstlane(threadIdx.x) >= THREADS / 2;
        other.init(second ? a : b, second ? lda : ldb, second ? rows_a : rows_b, count, second ? a_end : b_end);
        Half::init(second ? b : a, second ? ldb : lda, second ? rows_b : rows_a, count, second ? b_end : a_end, second ? THREADS / 2 : 0);
        this->safe = this->safe && other.safe;
        this->slow = rows_a < Half::W || rows_b < Half::W;
        if (this->slow) this->r0 = ((int)threadIdx.x - (second ? THREADS / 2 : 0)) / Half::BKC * Half::W;
    }
    __device__ __forceinline__ void store(const Regs &reg, char *lds) const { Half::store(reg, lds + (second ? ROWS * Half::BKC * 16 * T::PLANES : 0)); }
    __device__ __forceinline__ void add_up(const Regs &reg) { if (second) Half::add_up(reg); }
    __device__ __forceinline__ float total(float *lds) const { return Half::total(lds, second); }
};
// the other place
template <class T> struct Nothing {
    static constexpr int STEP = T::BKC * 8, N_LOADS = 0, N_STORES = 0;
    static constexpr bool slow = false, safe = true;
    struct Regs {};
    __device__ __forceinline__ void load(Regs &, int) const {}
    __device__ __forceinline__ void load_guarded(Regs &, int) const {}
    __device__ __forceinline__ void trim(Regs &, int) const {}
    __device__ __forceinline__ void store(const Regs &, char *) const {}
};

// ---- a shape of tile: BM rows by BN columns of C over WM x WN waves
template <class T_, int BM_, int BN_, int WM_, int WN_, int BUFFERS_ = 2, int DEPTH_ = 1> struct Shape {
    typedef T_ T;
    static constexpr int BUFFERS = BUFFERS_, DEPTH = DEPTH_;               // steps in LDS, and in registers (product())
    static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, THREADS = 64 * WM * WN;
    static constexpr int MI = BM / WM / 16, NI = BN / WN / 16;             // 16 x 16 results a wave
    static constexpr int A_BYTES = BN * T::BKC * 16 * T::PLANES, B_BYTES = BM * T::BKC * 16 * T::PLANES;
    static constexpr int RING = BM * BN == 65536 ? 5 : 4, LDS = T::PLANES == 1 ? RING * (A_BYTES + B_BYTES) / 2 : BUFFERS * (A_BYTES + B_BYTES);
    static constexpr bool ALONE = LDS > 80 << 10;                          // one workgroup a CU
    typedef typename T::acc Acc[MI][NI];
    // where a lane's results lie: rows row() + 16 m, columns col() + 16 n .. + 3
    static __device__ __forceinline__ int row() { return (int)(threadIdx.x >> 6) / WN * (BM / WM) + (int)(threadIdx.x & 15); }
    static __device__ __forceinline__ int col() { return (int)(threadIdx.x >> 6) % WN * (BN / WN) + 4 * ((int)(threadIdx.x & 63) >> 4); }
    static __device__ __forceinline__ int wave_col() { return (int)(threadIdx.x >> 6) % WN; }
    static __device__ __forceinline__ int wave_row() { return (int)(threadIdx.x >> 6) / WN; }
};

// ---- the core: acc[mi][ni] += A B^T over c = 0 .. count; A gives i (BN), B gives j (BM)
template <class S> struct Fragments {
    typedef typename S::T T;
    static constexpr int P = T::PLANES, BKC = T::BKC;
    static constexpr int N_READS = P * (S::NI + S::MI), N_MFMA = S::NI * S::MI * (P == 1 ? 1 : 6);
    u32x4 a[P][S::NI], b[P][S::MI];
    // chunks 4 s .. 4 s + 3 of the rows of this lane's operands
    __device__ __forceinline__ void read(const char *lds, int s)
    {
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, q = 4 * s + (lane >> 4);
        const char *pa = lds + wave % S::WN * (S::BN / S::WN * BKC * 16) + lds_at<BKC>(lane & 15, q);
        const char *pb = lds + S::A_BYTES + wave / S::WN * (S::BM / S::WM * BKC * 16) + lds_at<BKC>(lane & 15, q);
#pragma unroll
        for (int p = 0; p < P; ++p) {
#pragma unroll
            for (int n = 0; n < S::NI; ++n) a[p][n] = *reinterpret_cast<const u32x4 *>(pa + (p * S::BN + 16 * n) * (BKC * 16));
#pragma unroll
            for (int m = 0; m < S::MI; ++m) b[p][m] = *reinterpret_cast<const u32x4 *>(pb + (p * S::BM + 16 * m) * (BKC * 16));
        }
    }
    __device__ __forceinline__ void multiply(typename S::Acc &acc) const
    {
#pragma unroll
        for (int m = 0; m < S::MI; ++m)
#pragma unroll
            for (int n = 0; n < S::NI; ++n) {
                if constexpr (P == 1) {
                    acc[m][n] = T::mma(a[0][n], b[0][m], acc[m][n]);
                } else {                     // smallest first
                    acc[m][n] = T::mma(a[1][n], b[1][m], acc[m][n]);
                    acc[m][n] = T::mma(a[2][n], b[0][m], acc[m][n]);
                    acc[m][n] = T::mma(a[0][n], b[2][m], acc[m][n]);
                    acc[m][n] = T::mma(a[1][n], b[0][m], acc[m][n]);
                    acc[m][n] = T::mma(a[0][n], b[1][m], acc[m][n]);
                    acc[m][n] = T::mma(a[0][n], b[0][m], acc[m][n]);
                }
            }
    }
};

// Scheduling of one multiplication: each instruction of the other kinds is issued behind its share of matrix
// instructions, so that the matrix unit never waits for a run of them.
template <int MFMA, int READS, int STORES, int LOADS> __device__ __forceinline__ void interleave()
{
    // the last quarter of the matrix instructions covers the latency of the last read
    constexpr int OTHERS = READS + STORES + LOADS, BEHIND = MFMA * 3 / 4, EACH = OTHERS ? BEHIND / OTHERS : 0, MORE = OTHERS ? BEHIND % OTHERS : 0;
#pragma unroll
    for (int k = 0; k < OTHERS; ++k) {
        if (k < READS) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        else if (k < READS + STORES) __builtin_amdgcn_sched_group_barrier(0x200, 1, 0);
        else __builtin_amdgcn_sched_group_barrier(0x20, 1, 0);
        if (k < MORE) __builtin_amdgcn_sched_group_barrier(0x8, EACH + 1, 0);
        else if (EACH > 0) __builtin_amdgcn_sched_group_barrier(0x8, EACH, 0);
    }
}

template <class LA, class LB> __device__ __forceinline__ void add_up(LA &, typename LA::Regs &, LB &b, typename LB::Regs &rb) { b.add_up(rb); }
template <class LA, class T> __device__ __forceinline__ void add_up(LA &a, typename LA::Regs &ra, Nothing<T> &, typename Nothing<T>::Regs &) { a.add_up(ra); }

// While one step is multiplied, the next goes from registers to LDS and later ones are loaded: S::DEPTH sets of registers hold
// as many steps in flight (the last steps load themselves once more instead of branching: a branch around the loads makes the
// compiler wait for them at its end).
// Two buffers (one barrier a step, before its last multiplication): behind the barrier the next step lies in the other half of
// LDS, so that its first operands are read under that multiplication, and every wave has read the last of this step's, so that its
// half may be overwritten.  One buffer (two barriers a step): half the LDS, for two workgroups a CU that fill each other's waits.
// `sums`: add up B's rows over c as well (a Strided operand or a pair; workgroup-uniform).
template <class S, bool SUMS = false, class LA, class LB>
__device__ __forceinline__ void product(LA &a, LB &b, int count, char *lds, typename S::Acc &acc, bool sums = false)
{
    constexpr int STEP = LA::STEP, SUB = S::T::BKC / 4, HALF = S::A_BYTES + S::B_BYTES, D = S::DEPTH;
    static_assert(LA::STEP == LB::STEP, "one step for both operands");
    // whole steps, and the step that the loads end on: what is left behind them, if it may be read whole
    const int steps = a.slow || b.slow ? 0 : count / STEP, rest = count - count / STEP * STEP;
    const bool tail = rest > 0 && !a.slow && !b.slow && a.safe && b.safe;
    const int last = steps - 1 + (tail ? 1 : 0);
    typename LA::Regs ra[D];
    typename LB::Regs rb[D];
    if (last >= 0) {
        Fragments<S> f[2];
        auto load = [&](int k, int step) {
            const int c0 = min(step, last) * STEP;
            a.load(ra[k], c0);
            b.load(rb[k], c0);
        };
        // step `step` from registers to LDS
        auto store = [&](int k, int step, char *to) {
            if constexpr (SUMS)
                if (sums && step < steps) add_up(a, ra[k], b, rb[k]);
            a.store(ra[k], to);
            b.store(rb[k], to + S::A_BYTES);
        };
#pragma unroll
        for (int k = 0; k < D; ++k) load(k, k);
        if (steps > 0) {
            store(0, 0, lds);
            load(0, D);
            __syncthreads();
            int here = 0;
            if constexpr (SUB == 2 && S::BUFFERS == 2) f[0].read(lds, 0);
            for (int t0 = 0; t0 < steps; t0 += D) {
#pragma unroll
                for (int k = 0; k < D; ++k) {
                    const int t = t0 + k, set = (k + 1) % D;
                    if (k > 0 && t >= steps) break;
                    if constexpr (S::BUFFERS == 1) {
#pragma unroll
                        for (int s = 0; s < SUB; ++s) {
                            f[0].read(lds, s);
                            f[0].multiply(acc);
                        }
                        __syncthreads();
                        store(set, t + 1, lds);
                        load(set, t + 1 + D);
                        __syncthreads();
                    } else {
                        const int there = HALF - here;
                        f[1].read(lds + here, SUB - 1);
                        store(set, t + 1, lds + there);
                        load(set, t + 1 + D);
                        if constexpr (SUB == 2) {
                            f[0].multiply(acc);
                            interleave<Fragments<S>::N_MFMA, Fragments<S>::N_READS, LA::N_STORES + LB::N_STORES, LA::N_LOADS + LB::N_LOADS>();
                            __syncthreads();
                            f[0].read(lds + there, 0);
                            f[1].multiply(acc);
                            interleave<Fragments<S>::N_MFMA, Fragments<S>::N_READS, 0, 0>();
                        } else {
                            f[1].multiply(acc);
                            __syncthreads();
                        }
                        here = there;
                    }
                }
            }
            __syncthreads();
        }
        if (tail) {                          // every set of registers holds it by now
            a.trim(ra[0], last * STEP);
            b.trim(rb[0], last * STEP);
        }
    }
    // what is left of the last step, from where the loads above ended or through the guarded loads
    for (int c0 = steps * STEP; c0 < count; c0 += STEP) {
        Fragments<S> f;
        if (!tail) {
            a.load_guarded(ra[0], c0);
            b.load_guarded(rb[0], c0);
        }
        if constexpr (SUMS)
            if (sums) add_up(a, ra[0], b, rb[0]);
        a.store(ra[0], lds);
        b.store(rb[0], lds + S::A_BYTES);
        __syncthreads();
#pragma unroll
        for (int s = 0; s < SUB; ++s) {
            f.read(lds, s);
            f.multiply(acc);
        }
        __syncthreads();
    }
    if constexpr (S::T::PLANES == 3)
#pragma unroll
        for (int m = 0; m < S::MI; ++m)
#pragma unroll
            for (int n = 0; n < S::NI; ++n) acc[m][n] *= SPLIT_UNSCALE;
}

// ---- the way out: a wave turns 16 rows of its results through LDS (its own piece: no barrier) so that a lane holds 16 bytes
// of a row and a row's part of the tile leaves as whole lines; four results a lane, as the MFMA leaves them, are 8 bytes of
// 16 rows a store, and a tile of 256 x 256 took 15 us to leave that way.
template <class S, class E> struct Out {
    static constexpr int V = 16 / sizeof(E), COLS = S::NI * 16, LD = COLS + 4, LANES = COLS / V, ROWS = 64 / LANES, TURNS = 16 / ROWS;
    static_assert(S::WM * S::WN * 16 * LD * 4 <= S::LDS, "LDS");
    static __device__ __forceinline__ int col() { return S::wave_col() * COLS + (int)(threadIdx.x & 63) % LANES * V; }
    static __device__ __forceinline__ int row(int m, int t) { return S::wave_row() * (S::BM / S::WM) + 16 * m + t * ROWS + (int)(threadIdx.x & 63) / LANES; }
    // the values of block m at (row(m, t), col() ..), all t; `block(n)` gives the MFMA's four values of column block n
    template <class B> static __device__ __forceinline__ void turn(char *lds, float (&v)[TURNS][V], B block)
    {
        const int lane = threadIdx.x & 63;
        float *own = (float *)lds + (threadIdx.x >> 6) * (16 * LD);
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int n = 0; n < S::NI; ++n) wm_store4(own + (lane & 15) * LD + 16 * n + 4 * (lane >> 4), block(n));
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int t = 0; t < TURNS; ++t)
#pragma unroll
            for (int k = 0; k < V; k += 4) {
                const f32x4 f = wm_load4(own + (t * ROWS + lane / LANES) * LD + lane % LANES * V + k);
#pragma unroll
                for (int e = 0; e < 4; ++e) v[t][k + e] = f[e];
            }
        __builtin_amdgcn_wave_barrier();
    }
    // up to V consecutive elements
    template <class F> static __device__ __forceinline__ void load(const F *p, int have, float (&v)[V])
    {
        typedef F vec __attribute__((ext_vector_type(V), aligned(sizeof(F))));
        if (have >= V) {
            const vec x = *reinterpret_cast<const vec *>(p);
#pragma unroll
            for (int k = 0; k < V; ++k) v[k] = to_float((F)x[k]);
        } else {
#pragma unroll
            for (int k = 0; k < V; ++k) v[k] = k < have ? to_float(p[k]) : 0.0f;
        }
    }
    static __device__ __forceinline__ void store(E *p, int have, const float (&v)[V])
    {
        typedef E vec __attribute__((ext_vector_type(V), aligned(sizeof(E))));
        if (have >= V) {
            vec x;
#pragma unroll
            for (int k = 0; k < V; ++k) x[k] = from_float<E>(v[k]);
            *reinterpret_cast<vec *>(p) = x;
        } else {
#pragma unroll
            for (int k = 0; k < V; ++k)
                if (k < have) p[k] = from_float<E>(v[k]);
        }
    }
};

// The elements of C that are not finite once more, on the float32 MFMA from memory, by the wave that holds one (`cols` of i and `rows`
// of j count; element (i, c) of A at a + i ai + c ac).  Where all of them are NaN a launch takes 4 to 11 times as long; by a
// loop over c for each element it took 40 to 150 times as long.
template <class S>
__device__ __forceinline__ void not_finite_again(typename S::Acc &acc, const float *a, long long ai, long long ac, const float *b, long long bj,
                                                 long long bc, int cols, int rows, int count)
{
    const auto bad = [&](int m, int n, int k) {
        return !(fabsf(acc[m][n][k]) <= 3.4028235e38f) && S::col() + 16 * n + k < cols && S::row() + 16 * m < rows;
    };
    bool any = false;
#pragma unroll
    for (int m = 0; m < S::MI; ++m)
#pragma unroll
        for (int n = 0; n < S::NI; ++n)
#pragma unroll
            for (int k = 0; k < 4; ++k) any |= bad(m, n, k);
    if (__ballot(any) == 0) return;
    const int lane = threadIdx.x & 63, i0 = S::wave_col() * (S::BN / S::WN) + (lane & 15), j0 = S::row();
    // a row of blocks at a time, for the registers' sake
#pragma unroll
    for (int m = 0; m < S::MI; ++m) {
        f32x4 again[S::NI] = {};
        const float *bp = b + (long long)min(j0 + 16 * m, rows - 1) * bj;
#pragma unroll 2
        for (int c0 = 0; c0 < count; c0 += 4) {
            const int c = c0 + (lane >> 4), have = min(c, count - 1);
            const float y = c < count ? bp[have * bc] : 0.0f;
#pragma unroll
            for (int n = 0; n < S::NI; ++n) {
                const float x = a[min(i0 + 16 * n, cols - 1) * ai + have * ac];
                again[n] = __builtin_amdgcn_mfma_f32_16x16x4f32(c < count ? x : 0.0f, y, again[n], 0, 0, 0);
            }
        }
#pragma unroll
        for (int n = 0; n < S::NI; ++n)
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (bad(m, n, k)) acc[m][n][k] = again[n][k];
    }
}

// ---- ragged rows: group g owns rows offsets[g] .. offsets[g+1] - 1 of M.  Offsets outside 0 .. M are read as
// the nearest inside, one below an earlier one as that one, so any values give a partition of the rows.
// Rows that no group owns are the segments -1 (before offsets[0]) and G (behind offsets[G]).
struct Segment {
    int g, row0, rows;                       // group, first row and rows of a tile
    int parts;                               // tiles of the group
};

// a lane's value, in a scalar register
__device__ __forceinline__ int lane_value(int v, int lane) { return __builtin_amdgcn_readlane(v, lane); }

// Scans over the wave in data-parallel moves: 1, 2, 4 and 8 lanes up within rows of 16, then the rows' ends to the next row and the
// upper half (lanes without a source see `none`).
template <class F> __device__ __forceinline__ int wave_scan(int v, int none, F join)
{
    v = join(v, __builtin_amdgcn_update_dpp(none, v, 0x111, 0xF, 0xF, false));
    v = join(v, __builtin_amdgcn_update_dpp(none, v, 0x112, 0xF, 0xF, false));
    v = join(v, __builtin_amdgcn_update_dpp(none, v, 0x114, 0xF, 0xF, false));
    v = join(v, __builtin_amdgcn_update_dpp(none, v, 0x118, 0xF, 0xF, false));
    v = join(v, __builtin_amdgcn_update_dpp(none, v, 0x142, 0xA, 0xF, false));
    return join(v, __builtin_amdgcn_update_dpp(none, v, 0x143, 0xC, 0xF, false));
}
__device__ __forceinline__ int wave_scan(int v) { return wave_scan(v, 0, [](int a, int b) { return a + b; }); }

// Bounds of 64 segments s0 .. s0 + 63 in the lanes (segment s is group s - 1); `carry` is the bound before s0.
__device__ __forceinline__ void segment_bounds(const long long *offsets, int G, int M, int s0, int carry, int &lo, int &hi)
{
    const int s = s0 + (int)(threadIdx.x & 63);
    // the bound at the END of segment s: offsets[s] for s <= G, M behind
    long long v = s <= G ? (offsets ? offsets[s] : (s ? M : 0)) : M;
    int e = v < 0 ? 0 : v > M ? M : (int)v;
    hi = wave_scan(max(e, carry), 0, [](int a, int b) { return max(a, b); });
    lo = __builtin_amdgcn_update_dpp(carry, hi, 0x138, 0xF, 0xF, false);         // one lane up
}

// The map from the number of a tile of BM rows to its rows, built once a workgroup; what up to 62 groups need stays in the lanes.
struct RowTiles {
    const long long *offsets;
    int G, M, BM, lo, hi, total;             // bounds of the first 64 segments

    __device__ __forceinline__ RowTiles(const long long *offsets_, int G_, int M_, int BM_) : offsets(offsets_), G(G_), M(M_), BM(BM_), total(0)
    {
        int carry = 0;
        for (int s0 = 0; s0 < G + 2; s0 += 64) {
            int l, h;
            segment_bounds(offsets, G, M, s0, carry, l, h);
            if (s0 == 0) lo = l, hi = h;
            total += lane_value(wave_scan((h - l + BM - 1) / BM), 63);
            carry = lane_value(h, 63);
        }
    }
    __device__ __forceinline__ Segment tile(int t) const
    {
        int before = 0, carry = 0, l = lo, h = hi;
        for (int s0 = 0; s0 < G + 2; s0 += 64) {
            if (s0 > 0) segment_bounds(offsets, G, M, s0, carry, l, h);
            const int n = (h - l + BM - 1) / BM, upto = before + wave_scan(n);
            const uint64_t holds = __ballot(t < upto);
            if (holds) {
                const int k = __builtin_ctzll(holds);
                const int row0 = lane_value(l, k) + (t - lane_value(upto - n, k)) * BM;
                return {s0 + k - 1, row0, min(lane_value(h, k) - row0, BM), lane_value(n, k)};
            }
            before = lane_value(upto, 63);
            carry = lane_value(h, 63);
        }
        return {0, 0, 0, 0};
    }
    // the first tile of group g and how many it has
    __device__ __forceinline__ void tiles_of(int g, int &first, int &count) const
    {
        int before = 0, carry = 0, l = lo, h = hi;
        for (int s0 = 0;; s0 += 64) {
            if (s0 > 0) segment_bounds(offsets, G, M, s0, carry, l, h);
            const int n = (h - l + BM - 1) / BM, upto = before + wave_scan(n);
            if (g + 1 < s0 + 64) {
                count = lane_value(n, g + 1 - s0);
                first = lane_value(upto, g + 1 - s0) - count;
                return;
            }
            before = lane_value(upto, 63);
            carry = lane_value(h, 63);
        }
    }
};

// rows of group g (workgroup-uniform)
__device__ __forceinline__ void group_rows(const long long *offsets, int G, int M, int g, int &row0, int &rows)
{
    int carry = 0;
    for (int s0 = 0; s0 < G + 2; s0 += 64) {
        int lo, hi;
        segment_bounds(offsets, G, M, s0, carry, lo, hi);
        if (g + 1 < s0 + 64) {
            row0 = lane_value(lo, g + 1 - s0);
            rows = lane_value(hi, g + 1 - s0) - row0;
            return;
        }
        carry = lane_value(hi, 63);
    }
    row0 = rows = 0;
}

inline long long row_tiles_most(int G, int M, int BM)
{
    const long long n = (M + (long long)(G + 2) * (BM - 1)) / BM;
    return n < M ? n : M;                    // none is empty
}

// Workgroups go round the eight XCDs in turn: logical tiles are dealt out so that an XCD works on a run of
// them, and a run keeps to `band` row tiles and walks the columns, so that its operands stay in its L2 (us, row after row | so: 16384
// rows, 16 experts, gradients 4096 -> 2048 bf16 312 | 306; 2999 rows, 33 experts, gradients 333 -> 515 float16 21.7 | 19.4).
__device__ __forceinline__ void place_of_tile(int t, int row_tiles, int col_tiles, int band, int &rt, int &ct)
{
    const int total = row_tiles * col_tiles, per = total / 8, extra = total % 8, xcd = t % 8;
    const int id = xcd * per + min(xcd, extra) + t / 8;
    const int b = id / (band * col_tiles), in = id - b * band * col_tiles, height = min(band, row_tiles - b * band);
    rt = b * band + in % height;
    ct = in / height;
}

// The work of a workgroup: a tile of S, or part of one.  `slots` workgroups run at once; the tiles that are left when they
// have been filled a whole number of times are cut into tiles of Quarter or of Half where those find room at once, so that a
// launch ends after a part of a tile's time instead of a whole one (us, whole | cut: 8191 rows, 8 experts of 1024 -> 1024 float32 130 | 104,
// their gradients 159 | 124; 16384 rows, 16 experts, gradients 4096 -> 2048 bf16 344 | 306; int8 777 x 1283 -> 1001 23 | 15).  Halves
// only where a tile has a CU to itself: two tiles to a CU leave one each for half of the slots, which is as fast (45001 x 216 x 432
// float32 71 us whole, 76 in halves).
template <class S, class Half, class Quarter> struct Cut {
    typedef typename std::conditional<S::ALONE, Half, S>::type H;
    static_assert(S::THREADS == H::THREADS && H::LDS <= S::LDS && (!S::ALONE || S::BM * S::BN == 2 * H::BM * H::BN), "one launch");
    static_assert(S::THREADS == Quarter::THREADS && Quarter::LDS <= S::LDS && S::BM * S::BN == 4 * Quarter::BM * Quarter::BN, "one launch");
    int tile, row, col, parts;               // tile < 0: nothing; row and col of the part in it
    __device__ __forceinline__ Cut(int block, int total, int slots)
    {
        const int left = total % slots;
        parts = left * 4 <= slots ? 4 : S::ALONE && left * 2 <= slots ? 2 : 1;
        const int whole = parts > 1 ? total - left : total;
        if (block < whole) parts = 1;
        const int k = block < whole ? 0 : block - whole;
        tile = block < whole ? block : whole + k / parts;
        const int i = k % parts, across = parts == 4 ? S::BN / Quarter::BN : S::BN / H::BN;
        row = i / across * (parts == 4 ? Quarter::BM : H::BM);
        col = i % across * (parts == 4 ? Quarter::BN : H::BN);
        if (tile >= total) tile = -1;
    }
    static long long blocks(long long total_most, int slots) { return total_most + (long long)slots / 4 * 3; }
};

// The order in which the groups' products over rows are taken up: the longest first, so that a launch does not end on one of
// them; where two workgroups share a CU from the start (`first` groups are begun on empty CUs), the shortest are put beside the
// longest (38115 rows in 16 uneven experts, us, in order | so: 512 x 512 bf16 57 | 54, float32 170 | 166).  More than 62 groups are
// taken as they come.  Gives the group and its rows.
__device__ __forceinline__ void group_in_turn(const long long *offsets, int G, int M, int turn, int first, int &g, int &row0, int &rows)
{
    if (G > 62) {
        g = turn;
        group_rows(offsets, G, M, g, row0, rows);
        return;
    }
    int lo, hi;
    segment_bounds(offsets, G, M, 0, 0, lo, hi);
    const int lane = threadIdx.x & 63, size = hi - lo;
    int rank = 0;
    for (int j = 1; j <= G; ++j) {
        const int other = lane_value(size, j);
        rank += other > size || (other == size && j < lane) ? 1 : 0;
    }
    const int want = turn < first ? turn : G - 1 - (turn - first);
    const int k = __builtin_ctzll(__ballot(lane >= 1 && lane <= G && rank == want));
    g = k - 1;
    row0 = lane_value(lo, k);
    rows = lane_value(hi, k) - row0;
}

}  // namespace tile
