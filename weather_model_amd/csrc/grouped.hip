// grouped.hip -- Dense layers of several experts at once: rows sorted by expert, expert g owning rows
// offsets[g] .. offsets[g+1] - 1 of x (M, K) and its own weights W[g] (N, K) and bias b[g] (N).
//   forward   y[r][n]     = act(b[g][n] + sum_k x[r][k] W[g][n][k])
//   backward  gx[r][k]    = mask(sum_n gy[r][n] W[g][n][k])
//             gW[g][n][k] = sum_{r of g} gy[r][n] x[r][k],   gb[g][n] = sum_{r of g} gy[r][n]
// The number of rows of an expert is only known on the device, so a launch has as many workgroups as any
// partition of M rows can need tiles, and each finds its tile from the offsets (tile_gemm.h).
// Bound by the matrix unit where the experts have hundreds of rows (direct_gemm.h has the figures of 16 bits; float32, 8191 rows, 8
// experts of 1024 -> 1024: forward 107 us = 161 TFLOP/s, gx 132, gW 123, where a library float32 product of 8192^3 makes 155 and
// six bf16 products could make 227: splitting and LDS reads share the issue slots), by reading the weights where they have a few.
#include "direct_gemm.h"
#include "few_rows.h"

namespace {

using namespace tile;

constexpr int THREADS = 256;                 // of the kernels without tiles

// ---- rows: out (M, NO) = x (M, C) times W[g], forward (W[g] is (NO, C), its c along memory) or backward
// (W[g] is (C, NO)).  bias and relu are the forward's, mask the backward's.
// Of the contraction the C values from c0 on, of `depth`; out is of the type of x, or float32 for a part of the sums.
template <class S, bool BACKWARD, bool DIRECT, class E, class OUT>
__device__ __forceinline__ void rows_tile(const E *__restrict__ x, const E *__restrict__ W, const E *__restrict__ bias, const E *__restrict__ mask,
                                          OUT *__restrict__ out, char *lds, Segment s, int n0, int G, int M, int NO, int depth, int c0, int C,
                                          int relu)
{
    typedef typename S::T T;
    constexpr int BM = S::BM, BN = S::BN, THREADS = S::THREADS;
    s.rows = min(s.rows, BM);
    const int cols = min(BN, NO - n0);
    if (s.rows <= 0 || cols <= 0) return;
    if (s.g < 0 || s.g >= G) {                       // rows of no expert: zeros
        for (int e = threadIdx.x; e < s.rows * cols; e += THREADS) out[(long long)(s.row0 + e / cols) * NO + n0 + e % cols] = (OUT)0.0f;
        return;
    }
    const E *wg = W + (long long)s.g * NO * depth;
    const E *xr = x + (long long)s.row0 * depth + c0;
    const E *wt = BACKWARD ? wg + (long long)c0 * NO + n0 : wg + (long long)n0 * depth + c0;
    constexpr int MI = S::MI;
    typename S::Acc acc = {};
    if constexpr (DIRECT) {
        typename std::conditional<BACKWARD, DirectCols<T, BN, THREADS>, DirectRows<T, BN, THREADS>>::type a;
        DirectRows<T, BM, THREADS> b;
        a.init(wt, BACKWARD ? NO : depth, cols, C, W + (long long)G * NO * depth);
        b.init(xr, depth, s.rows, C, x + (long long)M * depth);
        product_direct<S, S::RING>(a, b, C, s.rows, lds, acc);
    } else {
        typename std::conditional<BACKWARD, Strided<T, BN, THREADS>, Contiguous<T, BN, THREADS>>::type a;
        Contiguous<T, BM, THREADS> b;
        a.init(wt, BACKWARD ? NO : depth, cols, C, W + (long long)G * NO * depth);
        b.init(xr, depth, s.rows, C, x + (long long)M * depth);
        product<S>(a, b, C, lds, acc);
    }

    if constexpr (T::PLANES == 3) not_finite_again<S>(acc, wt, BACKWARD ? 1 : depth, BACKWARD ? NO : 1, xr, depth, 1, cols, s.rows, C);
    typedef Out<S, OUT> O;
    const int col = O::col(), have = min(O::V, cols - col);
    if (S::wave_col() * O::COLS >= cols) return;
    float add[O::V] = {};
    if (!BACKWARD && bias) O::load(bias + (long long)s.g * NO + n0 + col, have, add);
    OUT *to = out + (long long)s.row0 * NO + n0 + col;
    const E *mk = mask ? mask + (long long)s.row0 * NO + n0 + col : nullptr;
#pragma unroll
    for (int m = 0; m < MI; ++m) {
        float v[O::TURNS][O::V], k[O::TURNS][O::V];
        if (BACKWARD && mk)
#pragma unroll
            for (int t = 0; t < O::TURNS; ++t)
                if (O::row(m, t) < s.rows) O::load(mk + (long long)O::row(m, t) * NO, have, k[t]);
        O::turn(lds, v, [&](int n) { return acc[m][n]; });
#pragma unroll
        for (int t = 0; t < O::TURNS; ++t) {
            if (O::row(m, t) >= s.rows) continue;
#pragma unroll
            for (int e = 0; e < O::V; ++e) {
                if (!BACKWARD) v[t][e] += add[e];
                if (!BACKWARD && relu) v[t][e] = relu_of(v[t][e]);
                if (BACKWARD && mk) v[t][e] = k[t][e] > 0.0f ? v[t][e] : 0.0f;
            }
            O::store(to + (long long)O::row(m, t) * NO, have, v[t]);
        }
    }
}

template <class S, class Half, class Quarter, bool BACKWARD, bool DIRECT, class E = typename S::T::elem>
__global__ __launch_bounds__(S::THREADS, 2) void grouped_rows_kernel(const E *__restrict__ x, const E *__restrict__ W, const E *__restrict__ bias,
                                                                  const E *__restrict__ mask, E *__restrict__ out,
                                                                  const long long *__restrict__ offsets, int G, int M, int NO, int C, int relu,
                                                                  int slots)
{
    __shared__ __attribute__((aligned(16))) char lds[S::LDS];
    const RowTiles tiles(offsets, G, M, S::BM);
    const int across = (NO + S::BN - 1) / S::BN;
    const Cut<S, Half, Quarter> cut(blockIdx.x, tiles.total * across, slots);
    if (cut.tile < 0) return;
    int rt, ct;
    place_of_tile(cut.tile, tiles.total, across, 8, rt, ct);
    Segment s = tiles.tile(rt);
    const int n0 = min(ct * S::BN, max(0, NO - S::BN));      // the last tile moves back over its neighbour
    s.row0 += cut.row;
    s.rows -= cut.row;
    if (cut.parts == 1) rows_tile<S, BACKWARD, DIRECT>(x, W, bias, mask, out, lds, s, n0, G, M, NO, C, 0, C, relu);
    else if (cut.parts == 4) rows_tile<Quarter, BACKWARD, DIRECT>(x, W, bias, mask, out, lds, s, n0 + cut.col, G, M, NO, C, 0, C, relu);
    else if constexpr (S::ALONE) rows_tile<Half, BACKWARD, DIRECT>(x, W, bias, mask, out, lds, s, n0 + cut.col, G, M, NO, C, 0, C, relu);
}

// Few tiles and a long contraction: blockIdx.y is a part of `depth` values of it, whose sums go to `partial`, (M, NO) each.
template <class S, bool BACKWARD, bool DIRECT, class E = typename S::T::elem>
__global__ __launch_bounds__(S::THREADS, 2) void grouped_rows_part_kernel(const E *__restrict__ x, const E *__restrict__ W, const E *__restrict__ bias,
                                                                       float *__restrict__ partial, const long long *__restrict__ offsets, int G, int M,
                                                                       int NO, int C, int depth)
{
    __shared__ __attribute__((aligned(16))) char lds[S::LDS];
    const RowTiles tiles(offsets, G, M, S::BM);
    const int across = (NO + S::BN - 1) / S::BN, c0 = blockIdx.y * depth;
    if ((int)blockIdx.x >= tiles.total * across) return;
    const int n0 = min((int)blockIdx.x % across * S::BN, max(0, NO - S::BN));      // the last tile moves back over its neighbour
    rows_tile<S, BACKWARD, DIRECT>(x, W, c0 == 0 ? bias : nullptr, (const E *)nullptr, partial + (long long)blockIdx.y * M * NO, lds,
                                   tiles.tile(blockIdx.x / across), n0, G, M, NO, C, c0, min(depth, C - c0), 0);
}
template <class E>
__global__ __launch_bounds__(THREADS) void grouped_rows_sum_kernel(const float *__restrict__ partial, const E *__restrict__ mask, E *__restrict__ out,
                                                                   long long count, int parts, int relu)
{
    const long long e = 4 * ((long long)blockIdx.x * THREADS + threadIdx.x);
    const int have = count - e < 4 ? (int)(count - e) : 4;
    if (have <= 0) return;
    f32x4 s = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int k = 0; k < parts; ++k) {
        const float *p = partial + k * count + e;
        if (have == 4) s += *reinterpret_cast<const Vec4<float>::type *>(p);
        else
            for (int i = 0; i < have; ++i) s[i] += p[i];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (relu) s[i] = relu_of(s[i]);
        if (mask && i < have) s[i] = to_float(mask[e + i]) > 0.0f ? s[i] : 0.0f;
    }
    if (have == 4) store4(out + e, s);
    else
        for (int i = 0; i < have; ++i) out[e + i] = from_float<E>(s[i]);
}

// ---- weights: gW[g] (N, K) = gy^T x over the rows of g: a workgroup takes a tile of one expert's, or with chunk > 0 of `chunk` rows of it.
// An expert of more than one chunk has them in `partial`, (N, K) each and (N) behind all of them, and
// grouped_weights_sum_kernel adds them in order.  gb is summed by the workgroups of the first columns from what is in LDS or in the
// registers that feed it.
template <class S, bool DIRECT, class E = typename S::T::elem>
__global__ __launch_bounds__(S::THREADS, 2) void grouped_weights_kernel(const E *__restrict__ gy, const E *__restrict__ x, E *__restrict__ gW,
                                                                     E *__restrict__ gb, float *__restrict__ partial, const long long *__restrict__ offsets, int G,
                                                                     int M, int N, int K, int chunk, int chunks, int first)
{
    typedef typename S::T T;
    constexpr int BM = S::BM, BN = S::BN, THREADS = S::THREADS;
    __shared__ __attribute__((aligned(16))) char lds[S::LDS];
    // i (contiguous in the output) is k, j is n
    const int kt = (K + BN - 1) / BN, nt = (N + BM - 1) / BM;
    int id = blockIdx.x;
    const int k0 = min(id % kt * BN, max(0, K - BN));       // last tiles move back over their neighbours
    id /= kt;
    const int n0 = min(id % nt * BM, max(0, N - BM));
    id /= nt;
    int g, row0, rows;
    float *own = nullptr, *own_bias = nullptr;               // where a part of an expert's sums goes
    if (chunk > 0) {
        const RowTiles map(offsets, G, M, chunk);
        if (id >= map.total) return;
        const Segment s = map.tile(id);
        if (s.g < 0 || s.g >= G) return;
        g = s.g, row0 = s.row0, rows = s.rows;
        if (s.parts > 1) {
            own = partial + (long long)id * N * K;
            own_bias = partial + (long long)chunks * N * K + (long long)id * N;
        }
    } else {
        group_in_turn(offsets, G, M, id, first, g, row0, rows);
    }
    constexpr int MI = S::MI;
    typename S::Acc acc = {};
    const int ks = min(BN, K), ns = min(BM, N);
    const E *xt = x + (long long)row0 * K + k0, *yt = gy + (long long)row0 * N + n0;
    const bool sums = gb && k0 == 0;
    auto bias = [&](int j, float v) {
        if (j >= ns) return;
        if (own) own_bias[n0 + j] = v;
        else gb[(long long)g * N + n0 + j] = from_float<E>(v);
    };
    if constexpr (DIRECT) {
        float sum[2] = {0.0f, 0.0f};
        if (rows > 0) {
            DirectCols<T, BN, THREADS> a;
            DirectCols<T, BM, THREADS> b;
            a.init(xt, K, ks, rows, nullptr);
            b.init(yt, N, ns, rows, nullptr);
            if (sums) product_direct<S, S::RING, true>(a, b, rows, ns, lds, acc, sum);
            else product_direct<S, S::RING>(a, b, rows, ns, lds, acc);
        }
        if (sums) {
            const float total = DirectCols<T, BM, THREADS>::total((float *)lds, sum);
            if ((int)threadIdx.x < BM) bias(threadIdx.x, total);
        }
    } else {
        float total = 0.0f;
        if (rows > 0) {
            static_assert(BM == BN, "a pair");
            StridedPair<T, BM, THREADS> pair;
            Nothing<T> none;
            pair.init(xt, K, ks, x + (long long)M * K, yt, N, ns, gy + (long long)M * N, rows);
            product<S, true>(pair, none, rows, lds, acc, sums);
            if (sums) total = pair.total((float *)lds);
        }
        if (sums && (int)threadIdx.x < BM) bias(threadIdx.x, total);
    }
    if constexpr (T::PLANES == 3) not_finite_again<S>(acc, xt, 1, K, yt, 1, N, ks, ns, rows);
    auto leave = [&](auto *to) {
        typedef Out<S, typename std::remove_pointer<decltype(to)>::type> O;
        const int col = O::col(), have = min(O::V, ks - col);
        if (S::wave_col() * O::COLS >= ks) return;
#pragma unroll
        for (int m = 0; m < MI; ++m) {
            float v[O::TURNS][O::V];
            O::turn(lds, v, [&](int n) { return acc[m][n]; });
#pragma unroll
            for (int t = 0; t < O::TURNS; ++t)
                if (O::row(m, t) < ns) O::store(to + (long long)O::row(m, t) * K + col, have, v[t]);
        }
    };
    __syncthreads();                                 // the bias sums have left LDS
    if (own) leave(own + (long long)n0 * K + k0);
    else leave(gW + ((long long)g * N + n0) * K + k0);
}

constexpr long long FEW_SUMS = 1 << 15;
// gW and gb of the experts that are in `partial` or have no rows; blockIdx.y is the expert.
template <class E>
__global__ __launch_bounds__(THREADS) void grouped_weights_sum_kernel(const float *__restrict__ partial, E *__restrict__ gW, E *__restrict__ gb,
                                                                      const long long *__restrict__ offsets, int G, int M, int N, long long count,
                                                                      int chunk, int chunks)
{
    const int g = blockIdx.y;
    int first, parts;
    RowTiles(offsets, G, M, chunk).tiles_of(g, first, parts);
    if (parts == 1) return;
    // `n` sums from p, `step` apart; the parts of small weights are shared out over the waves (100000 rows of 64 x 64 in 391 parts: 87 -> 46
    // us; 4096 rows of 432 x 216 in 16: 16 -> 21, not taken)
    __shared__ f32x4 join[4][64];
    const bool shared = parts > 8 && count <= FEW_SUMS;
    const int at = shared ? threadIdx.x & 63 : threadIdx.x, wave = shared ? threadIdx.x >> 6 : 0, waves = shared ? 4 : 1;
    const long long span = shared ? 256 : 4 * THREADS;
    const auto add = [&](const float *p, long long step, E *to, long long n) {
        for (long long e0 = span * blockIdx.x; e0 < n; e0 += span * gridDim.x) {
            const long long e = e0 + 4 * at;
            const int have = n - e < 4 ? (int)(n - e) : 4;
            f32x4 s = {0.0f, 0.0f, 0.0f, 0.0f};
            if (have == 4) {
#pragma unroll 8
                for (int k = wave; k < parts; k += waves) s += *reinterpret_cast<const Vec4<float>::type *>(p + k * step + e);
            } else {
                for (int k = wave; k < parts; k += waves)
                    for (int i = 0; i < have; ++i) s[i] += p[k * step + e + i];
            }
            if (shared) {
                join[wave][at] = s;
                __syncthreads();
                s = join[0][at];
                for (int w = 1; w < 4; ++w) s += join[w][at];
                __syncthreads();
            }
            if (wave == 0) {
                if (have == 4) store4(to + e, s);
                else
                    for (int i = 0; i < have; ++i) to[e + i] = from_float<E>(s[i]);
            }
        }
    };
    add(partial + first * count, count, gW + g * count, count);
    if (gb) add(partial + chunks * count + (long long)first * N, N, gb + (long long)g * N, N);
}

// ---- few rows: y (M, N) for groups of a handful of rows.  One read of the weights is the cost, so a workgroup takes 16
// outputs of one expert, its waves share the contraction, and the MFMA operands come straight from memory.
// Six waves a SIMD with four loads each of weights in flight (five for float32, whose operands are wider): 48 rows over 12 of 16
// experts of 2048 x 2048 bf16 in 22 us (4.5 TB/s from HBM); 28 with eight loads and four waves.
// Four waves in 16 bits, eight in float32 (us, four | eight, 8 rows of 8192 -> 8192 float32 85 | 68, of 2048 -> 8192 24 | 19; bf16 13.2 | 11.7,
// but 48 rows over the 12 experts 23 | 27).
template <class T, int WAVES>
__global__ __launch_bounds__(64 * WAVES, T::PLANES == 3 ? 5 : 6) void grouped_few_kernel(const typename T::elem *__restrict__ x, const typename T::elem *__restrict__ W,
                                                                   const typename T::elem *__restrict__ bias, typename T::elem *__restrict__ y,
                                                                   const long long *__restrict__ offsets, int G, int M, int N, int K, int relu)
{
    typedef typename T::elem E;
    __shared__ f32x4 part[WAVES][64];
    const int g = blockIdx.y, n0 = blockIdx.x * 16, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int row0, rows;
    if (g == G) {                                    // rows of no expert: zeros
        int end;
        group_rows(offsets, G, M, 0, row0, rows);
        group_rows(offsets, G, M, G - 1, end, rows);
        end += rows;
        const int cols = min(16, N - n0);
        for (int e = threadIdx.x; e < (row0 + M - end) * cols; e += 64 * WAVES) {
            const int r = e / cols;
            y[(long long)(r < row0 ? r : r - row0 + end) * N + n0 + e % cols] = (E)0.0f;
        }
        return;
    }
    group_rows(offsets, G, M, g, row0, rows);
    const E *wrow = W + ((long long)g * N + min(n0 + (lane & 15), N - 1)) * K;
    for (int r0 = 0; r0 < rows; r0 += 16) {
        const int r = min(r0 + (lane & 15), rows - 1);
        few::Dot<T, 2, WAVES> dot;
        dot.begin(wrow, W + (long long)G * N * K, K);
        const f32x4 acc = dot.multiply(few::RowOf<T>{x + (long long)(row0 + r) * K, x + (long long)M * K});
        if (wave > 0) part[wave][lane] = acc;
        __syncthreads();
        if (wave == 0) {
            f32x4 v = acc;
#pragma unroll
            for (int w = 1; w < WAVES; ++w) v += part[w][lane];
            const int n = n0 + 4 * (lane >> 4), have = min(4, N - n);
            if (r0 + (lane & 15) < rows && have > 0) {
                E *at = y + (long long)(row0 + r) * N + n;
                const E *b = bias ? bias + (long long)g * N + n : nullptr;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    if (b && k < have) v[k] += to_float(b[k]);
                    if (relu) v[k] = relu_of(v[k]);
                }
                if (have == 4) store4(at, v);
                else
                    for (int k = 0; k < have; ++k) at[k] = from_float<E>(v[k]);
            }
        }
        __syncthreads();
    }
}

int check(const char *who, int M, int N, int K, int G, int dtype)
{
    WM_REQUIRE(M >= 0 && N > 0 && K > 0 && G > 0, WM_ERR_INVALID, "%s: bad sizes M=%d N=%d K=%d groups=%d", who, M, N, K, G);
    WM_REQUIRE(N <= 1 << 20 && K <= 1 << 20 && G <= 4096 && M <= 1 << 30, WM_ERR_UNSUPPORTED,
               "%s: M=%d N=%d K=%d groups=%d is beyond 2^30 rows, 2^20 columns or 4096 groups", who, M, N, K, G);
    WM_REQUIRE(dtype == WM_F32 || dtype == WM_BF16 || dtype == WM_F16, WM_ERR_INVALID, "%s: bad dtype %d", who, dtype);
    WM_REQUIRE(wm_num_cus() > 0, WM_ERR_NO_DEVICE, "%s: no HIP device", who);
    return WM_OK;
}

int blocks_ok(const char *who, long long blocks)
{
    WM_REQUIRE(blocks <= (1ll << 32) / 512 - 1, WM_ERR_UNSUPPORTED, "%s: %lld tiles are too many for one launch", who, blocks);
    return WM_OK;
}

int workspace_ok(const char *who, size_t need, const void *workspace, size_t bytes)
{
    WM_REQUIRE(need == 0 || (workspace && bytes >= need), WM_ERR_WORKSPACE, "%s: workspace of %zu bytes needed, %zu given", who, need, bytes);
    WM_REQUIRE(need == 0 || ((uintptr_t)workspace & 15) == 0, WM_ERR_INVALID, "%s: workspace must be 16-byte aligned", who);
    return WM_OK;
}

template <class S, class Half, class Quarter, bool BACKWARD, bool DIRECT>
int rows_launch(const void *x, const void *W, const void *bias, const void *mask, void *out, const int64_t *offsets, int G, int M, int NO,
                int C, int relu, hipStream_t st)
{
    typedef typename S::T::elem E;
    const int slots = wm_num_cus() * (S::ALONE ? 1 : 2);
    const long long blocks = Cut<S, Half, Quarter>::blocks(row_tiles_most(G, M, S::BM) * ((NO + S::BN - 1) / S::BN), slots);
    if (int rc = blocks_ok("wm_dense_grouped", blocks)) return rc;
    hipLaunchKernelGGL((grouped_rows_kernel<S, Half, Quarter, BACKWARD, DIRECT>), dim3((unsigned)blocks), dim3(S::THREADS), 0, st, (const E *)x,
                       (const E *)W, (const E *)bias, (const E *)mask, (E *)out, (const long long *)offsets, G, M, NO, C, relu, slots);
    WM_LAUNCH_CHECK("grouped_rows_kernel");
    return WM_OK;
}

template <class T> struct Tiles {                       // 16-bit types
    typedef Shape<T, 256, 256, 2, 4> Large;
    typedef Shape<T, 128, 256, 2, 4> LargeHalf;
    typedef Shape<T, 128, 128, 2, 4> LargeQuarter;
    typedef Shape<T, 128, 128, 2, 2> Medium;
    typedef Shape<T, 64, 64, 2, 2, 2, 2> MediumQuarter;
};
template <> struct Tiles<F32> {
    typedef Shape<F32, 128, 128, 2, 2, 1> Medium;
    typedef Shape<F32, 64, 64, 2, 2, 1, 2> MediumQuarter;
};

// Values of the contraction that a workgroup takes where tiles of 64 x 64 are too few to hide a long one, or 0: whole.  us, whole | in parts,
// forward and backward: float32 1 expert, 100 rows of 1024 -> 1024 24 29 | 14 15, of 4096 82 99 | 25 28, 1024 rows of 4096 -> 1024 83
// 100 | 65 72, 16 experts, 200 rows of 2048 -> 256 43 52 | 20 22, 128 rows of 640 -> 8000 18 22 | 21 22 (not taken); 16 bits are
// quicker through a contraction: 6 experts, 1579 rows of 3599 -> 247 29 39 | 22 27, 100 rows of 4096 -> 1024 19 25 | 14 15, of 1024 10
// 11 | 13 15, 512 rows of 2048 -> 1024 11 15 | 14 15 (not taken).
int rows_depth(int G, int M, int NO, int C, int dtype)
{
    const bool f32 = dtype == WM_F32;
    const long long tiles = ((long long)M / 64 + (G < M ? G : M) / 2 + 1) * ((NO + 63) / 64);      // about
    if (C < (!f32 ? 2304 : tiles <= 256 ? 512 : 2048) || tiles > (f32 ? 512 : 256)) return 0;
    long long parts = tiles <= 256 ? 512 / tiles : 1024 / tiles;
    if (parts > (f32 ? 10 : 4)) parts = f32 ? 10 : 4;
    if (parts > C / (f32 ? 128 : 512)) parts = C / (f32 ? 128 : 512);
    return (int)wm_align_up((size_t)((C + parts - 1) / parts), 64);
}
size_t rows_bytes(int G, int M, int NO, int C, int dtype)
{
    const int depth = rows_depth(G, M, NO, C, dtype);
    return depth ? wm_align_up((size_t)((C + depth - 1) / depth) * M * NO * sizeof(float), 256) : 0;
}

template <class S, bool BACKWARD, bool DIRECT>
int rows_parts(const void *x, const void *W, const void *bias, const void *mask, void *out, float *partial, const int64_t *offsets, int G, int M,
               int NO, int C, int relu, int depth, hipStream_t st)
{
    typedef typename S::T::elem E;
    const long long blocks = row_tiles_most(G, M, S::BM) * ((NO + S::BN - 1) / S::BN), count = (long long)M * NO;
    const int parts = (C + depth - 1) / depth;
    if (int rc = blocks_ok("wm_dense_grouped", blocks * parts)) return rc;
    hipLaunchKernelGGL((grouped_rows_part_kernel<S, BACKWARD, DIRECT>), dim3((unsigned)blocks, parts), dim3(S::THREADS), 0, st, (const E *)x, (const E *)W,
                       (const E *)bias, partial, (const long long *)offsets, G, M, NO, C, depth);
    WM_LAUNCH_CHECK("grouped_rows_part_kernel");
    hipLaunchKernelGGL(grouped_rows_sum_kernel<E>, dim3((unsigned)((count + 4 * THREADS - 1) / (4 * THREADS))), dim3(THREADS), 0, st, (const float *)partial,
                       (const E *)mask, (E *)out, count, parts, relu);
    WM_LAUNCH_CHECK("grouped_rows_sum_kernel");
    return WM_OK;
}

// 16-byte rows go from memory to LDS, others through registers: 16384 rows, 8 experts of 1024 -> 1024 bf16 in tiles of 128 x 128, us,
// directly | through registers: forward 44 | 42, backward 43 | 79, gradients of weights 53 | 66.
template <class T, bool BACKWARD>
int rows_typed(const void *x, const void *W, const void *bias, const void *mask, void *out, void *workspace, const int64_t *offsets, int G, int M,
               int NO, int C, int relu, hipStream_t st)
{
    typedef Tiles<T> Z;
    const int depth = rows_depth(G, M, NO, C, std::is_same<T, F32>::value ? WM_F32 : WM_BF16);
    if constexpr (T::PLANES == 1) {
        if (direct_ok(x, 2ll * C) && direct_ok(W, BACKWARD ? 2ll * NO : 2ll * C)) {
            if (depth) return rows_parts<typename Z::MediumQuarter, BACKWARD, true>(x, W, bias, mask, out, (float *)workspace, offsets, G, M, NO, C, relu, depth, st);
            if (tiles_of_256(G, M, NO, wm_num_cus()))
                return rows_launch<typename Z::Large, typename Z::LargeHalf, typename Z::LargeQuarter, BACKWARD, true>(x, W, bias, mask, out, offsets, G, M, NO, C, relu, st);
            return rows_launch<typename Z::Medium, void, typename Z::MediumQuarter, BACKWARD, true>(x, W, bias, mask, out, offsets, G, M, NO, C, relu, st);
        }
    }
    if (depth) return rows_parts<typename Z::MediumQuarter, BACKWARD, false>(x, W, bias, mask, out, (float *)workspace, offsets, G, M, NO, C, relu, depth, st);
    return rows_launch<typename Z::Medium, void, typename Z::MediumQuarter, BACKWARD, false>(x, W, bias, mask, out, offsets, G, M, NO, C, relu, st);
}

// The few-rows kernel reads an expert's weights once for every 16 of its rows: it is for rows that are few even where one expert has
// them all, and in 16 bits not for long contractions, which tiles take in parts.  us, few rows | tiles, weights from HBM: bf16 1 expert, 8
// rows of 640 -> 8000 6.3 | 7.6, of 4096 -> 4096 17 | 13, 40 rows 38 | 14; 8 experts, 40 rows of 2048 -> 2048 18 | 27, 16 experts 37 | 35, 16
// experts, 8 rows of 4096 -> 1024 28 | 19; float32 1 expert, 8 rows of 640 -> 8000 8.7 | 14, of 4096 -> 4096 24 | 34, 16 experts, 40
// rows of 2048 -> 2048 68 | 71.
bool few_rows(int G, int M, int N, int K, int dtype)
{
    if (M > 16 && (M > 64 || G < 4)) return false;
    // rows of other than 16 bytes take the slower way into LDS
    return dtype == WM_F32 || K % 8 != 0 || rows_depth(G, M, N, K, dtype) == 0;
}

template <class T> int few_launch(const void *x, const void *W, const void *b, void *y, const int64_t *offsets, int G, int M, int N, int K,
                                  int relu, hipStream_t st)
{
    typedef typename T::elem E;
    constexpr int WAVES = T::PLANES == 3 ? 8 : 4;
    hipLaunchKernelGGL((grouped_few_kernel<T, WAVES>), dim3((N + 15) / 16, G + 1), dim3(64 * WAVES), 0, st, (const E *)x, (const E *)W, (const E *)b,
                       (E *)y, (const long long *)offsets, G, M, N, K, relu);
    WM_LAUNCH_CHECK("grouped_few_kernel");
    return WM_OK;
}

template <bool BACKWARD>
int rows_any(int dtype, const void *x, const void *W, const void *bias, const void *mask, void *out, void *workspace, const int64_t *offsets, int G,
             int M, int NO, int C, int relu, hipStream_t st)
{
    switch (dtype) {
    case WM_F32: return rows_typed<F32, BACKWARD>(x, W, bias, mask, out, workspace, offsets, G, M, NO, C, relu, st);
    case WM_BF16: return rows_typed<BF16, BACKWARD>(x, W, bias, mask, out, workspace, offsets, G, M, NO, C, relu, st);
    default: return rows_typed<F16, BACKWARD>(x, W, bias, mask, out, workspace, offsets, G, M, NO, C, relu, st);
    }
}

// Rows of a chunk, or 0 for whole experts: workgroups of 128 x 128 for two rounds of 256 CUs in float32, where a chunk takes long, and for
// one in 16 bits, and so many rows each that the sums of the chunks cost less.  Chunks are counted in rows and not in experts, as
// one expert may have most of the rows; experts of fewer than two chunks on average are cut only where they have twice the average.
// 432 -> 216, us with 1, 2, 4, 8, 16, 32 chunks an expert: bf16, 8 experts, 45000 rows 76 47 46 51 62 84 (taken: 4); float32 329 174
// 98 84 98 126 (8); with at least 128, 256, 512, 1024 rows: bf16, 1 expert, 4096 rows 19 15 16 21 (taken: 256), 17112 rows of 16 x 73 -> 116
// 15 15 20 28; float32 27 30 43 70 (128), 23 27 40 66.  Where the experts are enough, but one alone would be far from filling the card: 64
// experts, 45000 rows in one of them 2500 us whole in float32, 570 in bf16; 101 and 52 in chunks; evenly spread it costs the launch that
// finds nothing to add.  Layers of more tiles stay whole, whose parts would be as large as the weights for each chunk (all rows in one of 8
// experts of 1024 -> 1024 | evenly spread: 8192 rows float32 460 | 118, 16384 rows bf16 213 | 53; 16 experts of 2048 -> 4096 414 | 323).
int weight_chunk(int M, int N, int K, int G, int dtype)
{
    const int round = dtype == WM_F32 ? 512 : 256, least = dtype == WM_F32 ? 128 : 256;
    const long long tiles = (long long)((N + 127) / 128) * ((K + 127) / 128), want = (round + tiles - 1) / tiles;
    const bool enough = want <= G;
    if (M <= 2 * least || (enough && (tiles * 8 >= round || M < 32 * least))) return 0;
    const long long rows = enough || M / G < 2 * least ? 2ll * M / G : (M + want - 1) / want;
    return (int)wm_align_up((size_t)(rows < least ? least : rows), 64);
}
long long chunks_most(int G, int M, int chunk) { return chunk ? row_tiles_most(G, M, chunk) : 0; }

template <class S, bool DIRECT>
int weights_launch(const void *x, const void *gy, void *gW, void *gb, float *partial, const int64_t *offsets, int G, int M, int N, int K,
                   int chunk, hipStream_t st)
{
    typedef typename S::T::elem E;
    const long long chunks = chunks_most(G, M, chunk), blocks = (chunk ? chunks : G) * ((N + S::BM - 1) / S::BM) * ((K + S::BN - 1) / S::BN);
    if (int rc = blocks_ok("wm_dense_grouped_bwd_wb", blocks)) return rc;
    // experts begun on empty CUs, where all workgroups run at once
    const long long first = !chunk && blocks <= 2ll * wm_num_cus() && !S::ALONE ? wm_num_cus() / (blocks / G) : G;
    hipLaunchKernelGGL((grouped_weights_kernel<S, DIRECT>), dim3((unsigned)blocks), dim3(S::THREADS), 0, st, (const E *)gy, (const E *)x, (E *)gW,
                       (E *)gb, partial, (const long long *)offsets, G, M, N, K, chunk, (int)chunks, (int)first);
    WM_LAUNCH_CHECK("grouped_weights_kernel");
    return WM_OK;
}

template <class T>
int weights_typed(const void *x, const void *gy, void *gW, void *gb, void *workspace, const int64_t *offsets, int G, int M, int N, int K,
                  int chunk, hipStream_t st)
{
    typedef typename T::elem E;
    typedef typename Tiles<T>::Medium Md;
    float *partial = (float *)workspace;
    int rc;
    if constexpr (T::PLANES == 1) {
        typedef typename Tiles<T>::Large L;
        // 256 x 256 where they fill the CUs: 512 rows of 2048 -> 8192 31 -> 25 us, 16384 rows of 8 x 1024 -> 1024 (128 tiles) 53 -> 57
        const bool direct = direct_ok(x, 2ll * K) && direct_ok(gy, 2ll * N),
                   big = N >= 512 && K >= 512 && !chunk && (long long)G * (N / 256) * (K / 256) >= wm_num_cus();
        rc = direct && big ? weights_launch<L, true>(x, gy, gW, gb, partial, offsets, G, M, N, K, chunk, st)
             : direct      ? weights_launch<Md, true>(x, gy, gW, gb, partial, offsets, G, M, N, K, chunk, st)
                           : weights_launch<Md, false>(x, gy, gW, gb, partial, offsets, G, M, N, K, chunk, st);
    } else {
        rc = weights_launch<Md, false>(x, gy, gW, gb, partial, offsets, G, M, N, K, chunk, st);
    }
    if (rc != WM_OK || !chunk) return rc;
    const long long count = (long long)N * K;
    const long long many = (count + 1023) / 1024, grid = count <= FEW_SUMS ? (count + 255) / 256 : many > 1024 ? 1024 : many;
    hipLaunchKernelGGL(grouped_weights_sum_kernel<E>, dim3((unsigned)grid, G), dim3(THREADS), 0, st, (const float *)partial, (E *)gW, (E *)gb,
                       (const long long *)offsets, G, M, N, count, chunk, (int)chunks_most(G, M, chunk));
    WM_LAUNCH_CHECK("grouped_weights_sum_kernel");
    return WM_OK;
}

}  // namespace

extern "C" size_t wm_dense_grouped_fwd_workspace_bytes(int G, int M, int N, int K, int dtype)
{
    return M > 0 && N > 0 && K > 0 && G > 0 && !few_rows(G, M, N, K, dtype) ? rows_bytes(G, M, N, K, dtype) : 0;
}

extern "C" int wm_dense_grouped_fwd(const void *x, const void *W, const void *b, void *y, void *workspace, size_t workspace_bytes,
                                    const int64_t *offsets, int G, int M, int N, int K, int dtype, int relu, void *stream)
{
    if (int rc = check("wm_dense_grouped_fwd", M, N, K, G, dtype)) return rc;
    if (M == 0) return WM_OK;
    WM_REQUIRE(x && W && y && offsets, WM_ERR_INVALID, "wm_dense_grouped_fwd: null pointer");
    if (int rc = workspace_ok("wm_dense_grouped_fwd", wm_dense_grouped_fwd_workspace_bytes(G, M, N, K, dtype), workspace, workspace_bytes)) return rc;
    if (few_rows(G, M, N, K, dtype)) {
        hipStream_t st = (hipStream_t)stream;
        switch (dtype) {
        case WM_F32: return few_launch<F32>(x, W, b, y, offsets, G, M, N, K, relu, st);
        case WM_BF16: return few_launch<BF16>(x, W, b, y, offsets, G, M, N, K, relu, st);
        default: return few_launch<F16>(x, W, b, y, offsets, G, M, N, K, relu, st);
        }
    }
    return rows_any<false>(dtype, x, W, b, nullptr, y, workspace, offsets, G, M, N, K, relu, (hipStream_t)stream);
}

extern "C" size_t wm_dense_grouped_bwd_data_workspace_bytes(int G, int M, int N, int K, int dtype)
{
    return M > 0 && N > 0 && K > 0 && G > 0 ? rows_bytes(G, M, K, N, dtype) : 0;
}

extern "C" int wm_dense_grouped_bwd_data(const void *gy, const void *W, const void *mask_below, void *gx, void *workspace, size_t workspace_bytes,
                                         const int64_t *offsets, int G, int M, int N, int K, int dtype, void *stream)
{
    if (int rc = check("wm_dense_grouped_bwd_data", M, N, K, G, dtype)) return rc;
    if (M == 0) return WM_OK;
    WM_REQUIRE(gy && W && gx && offsets, WM_ERR_INVALID, "wm_dense_grouped_bwd_data: null pointer");
    if (int rc = workspace_ok("wm_dense_grouped_bwd_data", wm_dense_grouped_bwd_data_workspace_bytes(G, M, N, K, dtype), workspace, workspace_bytes))
        return rc;
    return rows_any<true>(dtype, gy, W, nullptr, mask_below, gx, workspace, offsets, G, M, K, N, 0, (hipStream_t)stream);
}

extern "C" size_t wm_dense_grouped_bwd_wb_workspace_bytes(int G, int M, int N, int K, int dtype)
{
    if (M < 0 || N <= 0 || K <= 0 || G <= 0) return 0;
    const int chunk = weight_chunk(M, N, K, G, dtype);
    return chunk ? wm_align_up((size_t)chunks_most(G, M, chunk) * N * (K + 1) * sizeof(float), 256) : 0;
}

extern "C" int wm_dense_grouped_bwd_wb(const void *x, const void *gy, void *gW, void *gb, void *workspace, size_t workspace_bytes,
                                       const int64_t *offsets, int G, int M, int N, int K, int dtype, void *stream)
{
    if (int rc = check("wm_dense_grouped_bwd_wb", M, N, K, G, dtype)) return rc;
    WM_REQUIRE((x && gy || M == 0) && gW && offsets, WM_ERR_INVALID, "wm_dense_grouped_bwd_wb: null pointer");
    if (int rc = workspace_ok("wm_dense_grouped_bwd_wb", wm_dense_grouped_bwd_wb_workspace_bytes(G, M, N, K, dtype), workspace, workspace_bytes)) return rc;
    const int chunk = weight_chunk(M, N, K, G, dtype);
    hipStream_t st = (hipStream_t)stream;
    switch (dtype) {
    case WM_F32: return weights_typed<F32>(x, gy, gW, gb, workspace, offsets, G, M, N, K, chunk, st);
    case WM_BF16: return weights_typed<BF16>(x, gy, gW, gb, workspace, offsets, G, M, N, K, chunk, st);
    default: return weights_typed<F16>(x, gy, gW, gb, workspace, offsets, G, M, N, K, chunk, st);
    }
}
