// int8.hip -- Dense layers served in 8 bits: codes with one scale per row (token) and per channel.
//   quantise  s_m = max_k |x[m][k]| / 127 (float32), q[m][k] = round(x[m][k] / s_m) to even, within +-127
//   product   y[m][n] = act((sum_k q[m][k] w[n][k]) s_m t_n + b[n]),  w (N, K) codes and t (N) scales of the weights
// The integer sum is exact (K <= 2^17 keeps it within 32 bits, -128 among the codes included); it is rounded
// to float32 once and scaled there.  A row of zeros has s = 0 and codes 0; a row that holds an infinity or a
// NaN has s = NaN and codes 0, so that all its outputs are NaN.
#include "direct_gemm.h"
#include "few_rows.h"

namespace {

using namespace tile;

// x / s rounded to even, as float32 division gives it.  x times the reciprocal is within 2^-22 of the quotient, relatively:
// only next to a tie (within 2^-15, |x / s| <= 128) can that round to another integer, and there it divides.
__device__ __forceinline__ float code_of(float x, float s, float r)
{
    const float t = x * r, n = rintf(t);
    if (fabsf(t - n) > 0.49996f) return rintf(x / s);
    return n;
}

// `LANES` threads a row, each NV vectors of 8 values in registers between the two passes; what does not fit (K > 8 LANES
// NV) is read again.  Codes go to q with row stride ldq >= K, zeros behind K.
template <class E, int LANES, int NV, int THREADS>
__device__ __forceinline__ void quantize_row(const E *__restrict__ row, int K, int8_t *to, long long ldq, float *scale)
{
    typedef E vec __attribute__((ext_vector_type(8), aligned(sizeof(E))));
    typedef uint32_t codes __attribute__((ext_vector_type(2), aligned(1)));
    __shared__ float part[THREADS / 64];
    const int t = threadIdx.x % LANES;
    auto load = [&](int k, float (&v)[8]) {
        if (k + 8 <= K) {
            const vec u = *reinterpret_cast<const vec *>(row + k);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = to_float((E)u[e]);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = k + e < K ? to_float(row[k + e]) : 0.0f;
        }
    };
    float v[NV][8], top = 0.0f;
    bool bad = false;
    auto see = [&](const float (&u)[8]) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float a = fabsf(u[e]);
            bad |= !(a <= 3.4028235e38f);
            top = fmaxf(top, a);
        }
    };
#pragma unroll
    for (int i = 0; i < NV; ++i) load(8 * (t + i * LANES), v[i]);
#pragma unroll
    for (int i = 0; i < NV; ++i) see(v[i]);
    for (int k = 8 * (t + NV * LANES); k < K; k += 8 * LANES) {
        float u[8];
        load(k, u);
        see(u);
    }
    if (bad) top = __builtin_inff();         // fmaxf drops a NaN: an infinity stands for both
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
    if constexpr (LANES == THREADS) {
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = top;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < THREADS / 64; ++w) top = fmaxf(top, part[w]);
    }
    const float s = top > 3.4028235e38f ? __builtin_nanf("") : top / 127.0f;
    const float r = s > 0.0f ? 1.0f / s : 0.0f;
    const bool far = r > 3.4028235e38f;      // a subnormal scale has no reciprocal
    auto put = [&](int k, const float (&u)[8]) {
        uint32_t w[2] = {0u, 0u};
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            float c = 0.0f;
            if (s > 0.0f) c = far ? rintf(u[e] / s) : code_of(u[e], s, r);
            c = fminf(fmaxf(c, -127.0f), 127.0f);
            w[e / 4] |= (uint32_t)(uint8_t)(int8_t)c << (8 * (e % 4));
        }
        if (k + 8 <= ldq) *reinterpret_cast<codes *>(to + k) = codes{w[0], w[1]};
        else
            for (int e = 0; e < 8 && k + e < ldq; ++e) to[k + e] = (int8_t)(w[e / 4] >> (8 * (e % 4)));
    };
#pragma unroll
    for (int i = 0; i < NV; ++i)
        if (8 * (t + i * LANES) < ldq) put(8 * (t + i * LANES), v[i]);
    for (int k = 8 * (t + NV * LANES); k < ldq; k += 8 * LANES) {
        float u[8];
        load(k, u);
        put(k, u);
    }
    if (t == 0) *scale = s;
}

template <class E, int LANES, int NV, int THREADS>
__global__ __launch_bounds__(THREADS) void quantize_rows_kernel(const E *__restrict__ x, int M, int K, int8_t *__restrict__ q, long long ldq,
                                                                float *__restrict__ scale)
{
    const int m = blockIdx.x * (THREADS / LANES) + threadIdx.x / LANES;
    if (LANES == 64 && m >= M) return;       // whole waves
    quantize_row<E, LANES, NV, THREADS>(x + (long long)m * K, K, q + m * ldq, ldq, scale + m);
}

template <class E, class S, bool DIRECT>
__device__ __forceinline__ void i8_tile(const int8_t *__restrict__ q, long long ldq, const float *__restrict__ qscale,
                                        const int8_t *__restrict__ W, const float *__restrict__ wscale, const float *__restrict__ bias,
                                        E *__restrict__ y, char *lds, Segment s, int n0, int G, int M, int N, int K, int relu)
{
    constexpr int BM = S::BM, BN = S::BN, THREADS = S::THREADS;
    s.rows = min(s.rows, BM);
    const int cols = min(BN, N - n0);
    if (s.rows <= 0 || cols <= 0) return;
    if (s.g < 0 || s.g >= G) {                       // rows of no expert: zeros
        for (int e = threadIdx.x; e < s.rows * cols; e += THREADS) y[(long long)(s.row0 + e / cols) * N + n0 + e % cols] = (E)0.0f;
        return;
    }
    typedef typename std::conditional<DIRECT, DirectRows<I8, BN, THREADS>, Contiguous<I8, BN, THREADS>>::type LA;
    typedef typename std::conditional<DIRECT, DirectRows<I8, BM, THREADS>, Contiguous<I8, BM, THREADS>>::type LB;
    LA a;
    LB b;
    a.init(W + ((long long)s.g * N + n0) * K, K, cols, K, W + (long long)G * N * K);
    b.init(q + s.row0 * ldq, ldq, s.rows, K, q + M * ldq);
    constexpr int MI = S::MI;
    typename S::Acc acc = {};
    if constexpr (DIRECT) product_direct<S, S::RING>(a, b, K, s.rows, lds, acc);
    else product<S>(a, b, K, lds, acc);
    // the compiler would convert the sums to float in the loop, on every turn
#pragma unroll
    for (int m = 0; m < MI; ++m)
#pragma unroll
        for (int n = 0; n < S::NI; ++n) asm volatile("" : "+v"(acc[m][n]));
    typedef Out<S, E> O;
    const int col = O::col(), have = min(O::V, cols - col);
    if (S::wave_col() * O::COLS >= cols) return;
    float ws[O::V], add[O::V];
    const long long c = (long long)s.g * N + n0 + col;
#pragma unroll
    for (int e = 0; e < O::V; ++e) {
        ws[e] = e < have ? wscale[c + e] : 0.0f;
        add[e] = bias && e < have ? bias[c + e] : 0.0f;
    }
    E *to = y + (long long)s.row0 * N + n0 + col;
#pragma unroll
    for (int m = 0; m < MI; ++m) {
        float v[O::TURNS][O::V], qs[O::TURNS];
#pragma unroll
        for (int t = 0; t < O::TURNS; ++t) qs[t] = qscale[s.row0 + min(O::row(m, t), s.rows - 1)];
        O::turn(lds, v, [&](int n) { return __builtin_convertvector(acc[m][n], f32x4); });
#pragma unroll
        for (int t = 0; t < O::TURNS; ++t) {
            if (O::row(m, t) >= s.rows) continue;
#pragma unroll
            for (int e = 0; e < O::V; ++e) {
                v[t][e] = v[t][e] * qs[t] * ws[e] + add[e];
                if (relu) v[t][e] = relu_of(v[t][e]);
            }
            O::store(to + (long long)O::row(m, t) * N, have, v[t]);
        }
    }
}

template <class E, class S, class Half, class Quarter, bool DIRECT>
__global__ __launch_bounds__(S::THREADS, 2) void dense_i8_kernel(const int8_t *__restrict__ q, long long ldq, const float *__restrict__ qscale,
                                                              const int8_t *__restrict__ W, const float *__restrict__ wscale,
                                                              const float *__restrict__ bias, E *__restrict__ y,
                                                              const long long *__restrict__ offsets, int G, int M, int N, int K, int relu, int slots)
{
    __shared__ __attribute__((aligned(16))) char lds[S::LDS];
    const RowTiles tiles(offsets, G, M, S::BM);
    const int across = (N + S::BN - 1) / S::BN;
    const Cut<S, Half, Quarter> cut(blockIdx.x, tiles.total * across, slots);
    if (cut.tile < 0) return;
    int rt, ct;
    place_of_tile(cut.tile, tiles.total, across, 8, rt, ct);
    Segment s = tiles.tile(rt);
    const int n0 = min(ct * S::BN, max(0, N - S::BN));       // the last tile moves back over its neighbour
    s.row0 += cut.row;
    s.rows -= cut.row;
    if (cut.parts == 1) i8_tile<E, S, DIRECT>(q, ldq, qscale, W, wscale, bias, y, lds, s, n0, G, M, N, K, relu);
    else if (cut.parts == 4) i8_tile<E, Quarter, DIRECT>(q, ldq, qscale, W, wscale, bias, y, lds, s, n0 + cut.col, G, M, N, K, relu);
    else if constexpr (S::ALONE) i8_tile<E, Half, DIRECT>(q, ldq, qscale, W, wscale, bias, y, lds, s, n0 + cut.col, G, M, N, K, relu);
}

// ---- few rows: one read of the weights (few_rows.h)
// joins the waves' sums; wave 0 scales and writes columns n0 .. n0 + 15 of row y (lane & 15), if `there`
template <int WAVES, class E>
__device__ __forceinline__ void few_out(i32x4 acc, i32x4 (&part)[WAVES][64], E *y, bool there, float qs, const float *wscale, const float *bias,
                                        int n0, int N, int relu)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (wave > 0) part[wave][lane] = acc;
    __syncthreads();
    if (wave == 0) {
#pragma unroll
        for (int w = 1; w < WAVES; ++w) acc += part[w][lane];
        const int n = n0 + 4 * (lane >> 4), have = min(4, N - n);
        if (there && have > 0) {
            f32x4 v;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int kk = n + min(k, have - 1);
                v[k] = (float)acc[k] * qs * wscale[kk] + (bias ? bias[kk] : 0.0f);
                if (relu) v[k] = relu_of(v[k]);
            }
            if (have == 4) store4(y + n, v);
            else
                for (int k = 0; k < have; ++k) y[n + k] = from_float<E>(v[k]);
        }
    }
    __syncthreads();
}

// zeros in columns n0 .. n0 + 15 of the rows of no expert
template <class E> __device__ __forceinline__ void few_zeros(E *y, const long long *offsets, int G, int M, int N, int n0)
{
    int row0, rows, end;
    group_rows(offsets, G, M, 0, row0, rows);
    group_rows(offsets, G, M, G - 1, end, rows);
    end += rows;
    const int cols = min(16, N - n0);
    for (int e = threadIdx.x; e < (row0 + M - end) * cols; e += blockDim.x) {
        const int r = e / cols;
        y[(long long)(r < row0 ? r : r - row0 + end) * N + n0 + e % cols] = (E)0.0f;
    }
}

constexpr int FEW_WAVES = 4;
template <class E>
__global__ __launch_bounds__(64 * FEW_WAVES) void dense_i8_few_kernel(const int8_t *__restrict__ q, long long ldq, const float *__restrict__ qscale,
                                                                    const int8_t *__restrict__ W, const float *__restrict__ wscale,
                                                                    const float *__restrict__ bias, E *__restrict__ y,
                                                                    const long long *__restrict__ offsets, int G, int M, int N, int K, int relu)
{
    __shared__ i32x4 part[FEW_WAVES][64];
    const int g = blockIdx.y, n0 = blockIdx.x * 16, lane = threadIdx.x & 63;
    if (g == G) return few_zeros(y, offsets, G, M, N, n0);
    int row0 = 0, rows = M;
    if (offsets) group_rows(offsets, G, M, g, row0, rows);
    const int8_t *wrow = W + ((long long)g * N + min(n0 + (lane & 15), N - 1)) * K;
    for (int r0 = 0; r0 < rows; r0 += 16) {
        const int r = row0 + min(r0 + (lane & 15), rows - 1);
        few::Dot<I8, 4, FEW_WAVES> dot;
        dot.begin(wrow, W + (long long)G * N * K, K);
        const i32x4 acc = dot.multiply(few::RowOf<I8>{q + r * ldq, q + M * ldq});
        few_out(acc, part, y + (long long)r * N, r0 + (lane & 15) < rows, qscale[r], wscale + (long long)g * N, bias ? bias + (long long)g * N : nullptr,
                n0, N, relu);
    }
}

// A few short rows: every workgroup makes their codes itself, in LDS, while its first weights are on their way -- the same codes as
// quantize_rows_kernel's, without its launch.  ONE: the whole workgroup takes the one row, K <= 8192; otherwise a wave takes a row.
// Eight waves for one row (us in a captured graph, four | eight waves: 4096 x 4096 10.1 | 7.8) and for five to eight (8 x 1024 x 4096 8.4 |
// 7.0), four for two to four (4 x 1024 x 4096 5.7 | 6.7).
constexpr int OWN_ROWS = 8, OWN_BYTES = 8192, OWN_LDS = OWN_BYTES + OWN_ROWS * 144;
struct Codes {                               // in LDS, zeros behind the row
    const int8_t *q;
    __device__ __forceinline__ u32x4 whole(int c) const { return *reinterpret_cast<const u32x4 *>(q + c); }
    __device__ __forceinline__ u32x4 part(int c, int) const { return whole(c); }
};

template <class E, bool ONE, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void dense_i8_own_kernel(const E *__restrict__ x, const int8_t *__restrict__ W,
                                                                    const float *__restrict__ wscale, const float *__restrict__ bias,
                                                                    E *__restrict__ y, const long long *__restrict__ offsets, int G, int M, int N,
                                                                    int K, int relu)
{
    __shared__ i32x4 part[WAVES][64];
    __shared__ __attribute__((aligned(16))) int8_t codes[OWN_LDS];
    __shared__ float scales[OWN_ROWS];
    const int g = blockIdx.y, n0 = blockIdx.x * 16, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (g == G) return few_zeros(y, offsets, G, M, N, n0);
    int row0 = 0, rows = M;
    if (offsets) group_rows(offsets, G, M, g, row0, rows);
    if (rows == 0) return;
    few::Dot<I8, 4, WAVES, true> dot;
    dot.begin(W + ((long long)g * N + min(n0 + (lane & 15), N - 1)) * K, W + (long long)G * N * K, K);
    const int ldq = (K + 127) / 128 * 128, stride = ldq + 16;        // 16: the rows' chunks in different banks
    if constexpr (ONE) {
        quantize_row<E, 64 * WAVES, OWN_BYTES / 8 / (64 * WAVES), 64 * WAVES>(x, K, codes, ldq, scales);
    } else {
        for (int r = wave; r < rows; r += WAVES)
            quantize_row<E, 64, 2048 / 8 / 64, 64 * WAVES>(x + (long long)(row0 + r) * K, K, codes + r * stride, ldq, scales + r);
    }
    __syncthreads();
    const int r = min(lane & 15, rows - 1);
    const i32x4 acc = dot.multiply(Codes{codes + r * stride});
    few_out(acc, part, y + (long long)(row0 + r) * N, (lane & 15) < rows, scales[r], wscale + (long long)g * N,
            bias ? bias + (long long)g * N : nullptr, n0, N, relu);
}

// Every 16 columns make the codes again: for rows whose codes take little more than the launch that this saves.  The choice is by the time
// of a call; in a captured graph it is within 0.1 us of the other or better.  us a call | in a captured graph, float32, codes here /
// in a launch of their own: 1 x 640 x 8000 8.3 / 12.7 | 6.3 / 6.7, 1 x 4096 x 4096 8.2 / 12.6 | 6.0 / 7.7, 2 x 2048 x 4096 8.3 / 12.5 | 6.1 /
// 6.0, 3 and 4 x 2048 x 4096 8.3 / 12.6 | 6.3 / 6.2, 4 x 1024 x 4096 8.3 / 12.7 | 5.3 / 6.2, 8 x 1024 x 4096 8.4 / 12.9 | 6.6 / 6.5, 8 x 640 x
// 8000 (four waves) 10.5 / 12.7 | 10.2 / 7.8 (not taken).
bool own_codes(int M, int N, int K)
{
    if (M == 1) return K <= OWN_BYTES;
    return (M <= 4 ? K <= 2048 : M <= OWN_ROWS && K <= 1024) && (long long)M * K * ((N + 4095) / 4096) <= OWN_BYTES;
}

size_t padded(int K) { return wm_align_up((size_t)K, 128); }

int check(const char *who, int M, int K, int dtype)
{
    WM_REQUIRE(M >= 0 && K > 0, WM_ERR_INVALID, "%s: bad sizes M=%d K=%d", who, M, K);
    WM_REQUIRE(K <= 1 << 17, WM_ERR_UNSUPPORTED, "%s: K=%d is beyond 2^17 (the integer sums would leave 32 bits)", who, K);
    WM_REQUIRE(M <= 1 << 24, WM_ERR_UNSUPPORTED, "%s: M=%d is beyond 2^24 rows", who, M);
    WM_REQUIRE(dtype == WM_F32 || dtype == WM_BF16 || dtype == WM_F16, WM_ERR_INVALID, "%s: bad dtype %d", who, dtype);
    WM_REQUIRE(wm_num_cus() > 0, WM_ERR_NO_DEVICE, "%s: no HIP device", who);
    return WM_OK;
}

// A wave a row up to 2048 values, a workgroup beyond.  With few rows the time is one row's chain of load, maximum and codes, and a row
// is spread over as many threads as leave each a vector.  us, bf16: 8192 rows of 4096 22 (4.7 TB/s; by single values 54); a
// wave | a workgroup a row: 16384 x 640 12 | 22, 16384 x 2048 24 | 28, 1000 x 640 4.2 | 3.6, 2000 x 2048 6.8 | 5.7; 200 x 8192 by
// 256 | 1024 threads 6.2 | 4.2.
template <class E> int quantize(const void *x, int M, int K, int8_t *q, long long ldq, float *scale, hipStream_t st)
{
#define WM_QUANTIZE(LANES, NV, THREADS)                                                                                                 \
    hipLaunchKernelGGL((quantize_rows_kernel<E, LANES, NV, THREADS>), dim3((M + THREADS / LANES - 1) / (THREADS / LANES)), dim3(THREADS), \
                       0, st, (const E *)x, M, K, q, ldq, scale)
    const int cus = wm_num_cus();
    if (M < 4 * cus && K > 4096) WM_QUANTIZE(1024, 1, 1024);
    else if (M < 4 * cus && K > 2048) WM_QUANTIZE(512, 1, 512);
    else if (M < (K > 1024 ? 16 : 4) * cus && K <= 2048) WM_QUANTIZE(256, 1, 256);
    else if (K <= 512) WM_QUANTIZE(64, 1, 256);
    else if (K <= 1024) WM_QUANTIZE(64, 2, 256);
    else if (K <= 2048) WM_QUANTIZE(64, 4, 256);
    else if (K <= 4096) WM_QUANTIZE(256, 2, 256);
    else WM_QUANTIZE(256, 4, 256);
#undef WM_QUANTIZE
    WM_LAUNCH_CHECK("quantize_rows_kernel");
    return WM_OK;
}

template <class E, class S, class Half, class Quarter, bool DIRECT>
int dense_tiles(const int8_t *q, long long ldq, const float *scale, const int8_t *W, const float *wscale, const float *b, void *y,
                const int64_t *offsets, int G, int M, int N, int K, int relu, hipStream_t st)
{
    const int slots = wm_num_cus() * (S::ALONE ? 1 : 2);
    const long long blocks = Cut<S, Half, Quarter>::blocks(row_tiles_most(G, M, S::BM) * ((N + S::BN - 1) / S::BN), slots);
    WM_REQUIRE(blocks <= (1ll << 32) / 512 - 1, WM_ERR_UNSUPPORTED, "wm_dense_i8: %lld tiles are too many for one launch", blocks);
    hipLaunchKernelGGL((dense_i8_kernel<E, S, Half, Quarter, DIRECT>), dim3((unsigned)blocks), dim3(S::THREADS), 0, st, q, ldq, scale, W, wscale, b, (E *)y,
                       (const long long *)offsets, G, M, N, K, relu, slots);
    WM_LAUNCH_CHECK("dense_i8_kernel");
    return WM_OK;
}

// As in grouped.hip, but for experts that fill the card with tiles.  us, few rows | tiles, weights from HBM: 1 expert, 16 rows of 4096 -> 4096
// 12 | 20, 40 rows of 8192 -> 8192 50 | 34; 8 experts, 40 rows of 2048 -> 2048 14 | 19, 16 experts 23 | 21, of 1024 -> 4096 39 | 22.
bool few_rows(int G, int M, int N, int K)
{
    if (M > 16 && (M > 64 || G < 4)) return false;
    return G == 1 || K % 16 != 0 || (long long)(G < M ? G : M) * N < 128 * 256;
}

template <class E>
int dense(const void *x, const int8_t *W, const float *wscale, const float *b, void *y, const int64_t *offsets, int G, int M, int N, int K, int relu,
          void *workspace, hipStream_t st)
{
    if (own_codes(M, N, K)) {
        const auto kernel = M == 1 ? dense_i8_own_kernel<E, true, 8> : M <= 4 ? dense_i8_own_kernel<E, false, 4> : dense_i8_own_kernel<E, false, 8>;
        hipLaunchKernelGGL(kernel, dim3((N + 15) / 16, offsets ? G + 1 : 1), dim3(M > 1 && M <= 4 ? 256 : 512), 0, st, (const E *)x, W, wscale, b,
                           (E *)y, (const long long *)offsets, G, M, N, K, relu);
        WM_LAUNCH_CHECK("dense_i8_own_kernel");
        return WM_OK;
    }
    float *scale = (float *)workspace;
    int8_t *q = (int8_t *)workspace + wm_align_up((size_t)M * sizeof(float), 256);
    const long long ldq = (long long)padded(K);
    if (int rc = quantize<E>(x, M, K, q, ldq, scale, st)) return rc;
    if (few_rows(G, M, N, K)) {
        hipLaunchKernelGGL(dense_i8_few_kernel<E>, dim3((N + 15) / 16, offsets ? G + 1 : 1), dim3(64 * FEW_WAVES), 0, st, q, ldq, scale, W, wscale, b,
                           (E *)y, (const long long *)offsets, G, M, N, K, relu);
        WM_LAUNCH_CHECK("dense_i8_few_kernel");
        return WM_OK;
    }
    typedef Shape<I8, 128, 128, 2, 2> Medium;
    typedef Shape<I8, 64, 64, 2, 2, 2, 2> MediumQuarter;
    if (direct_ok(W, K)) {
        if (tiles_of_256(G, M, N, wm_num_cus()))
            return dense_tiles<E, Shape<I8, 256, 256, 2, 4>, Shape<I8, 128, 256, 2, 4>, Shape<I8, 128, 128, 2, 4>, true>(
                q, ldq, scale, W, wscale, b, y, offsets, G, M, N, K, relu, st);
        return dense_tiles<E, Medium, void, MediumQuarter, true>(q, ldq, scale, W, wscale, b, y, offsets, G, M, N, K, relu, st);
    }
    return dense_tiles<E, Medium, void, MediumQuarter, false>(q, ldq, scale, W, wscale, b, y, offsets, G, M, N, K, relu, st);
}

}  // namespace

extern "C" int wm_quantize_rows_i8(const void *x, int M, int K, int dtype, int8_t *q, float *scale, void *stream)
{
    if (int rc = check("wm_quantize_rows_i8", M, K, dtype)) return rc;
    if (M == 0) return WM_OK;
    WM_REQUIRE(x && q && scale, WM_ERR_INVALID, "wm_quantize_rows_i8: null pointer");
    hipStream_t st = (hipStream_t)stream;
    switch (dtype) {
    case WM_F32: return quantize<float>(x, M, K, q, K, scale, st);
    case WM_BF16: return quantize<bf16_t>(x, M, K, q, K, scale, st);
    default: return quantize<f16_t>(x, M, K, q, K, scale, st);
    }
}

extern "C" size_t wm_dense_i8_workspace_bytes(int M, int N, int K)
{
    if (M <= 0 || N <= 0 || K <= 0 || own_codes(M, N, K)) return 0;
    return wm_align_up((size_t)M * sizeof(float), 256) + (size_t)M * padded(K);
}

extern "C" int wm_dense_i8(const void *x, const int8_t *W, const float *wscale, const float *b, void *y, const int64_t *offsets, int G, int M,
                           int N, int K, int dtype, int relu, void *workspace, size_t workspace_bytes, void *stream)
{
    if (int rc = check("wm_dense_i8", M, K, dtype)) return rc;
    WM_REQUIRE(N > 0 && G > 0, WM_ERR_INVALID, "wm_dense_i8: bad sizes N=%d groups=%d", N, G);
    WM_REQUIRE(offsets || G == 1, WM_ERR_INVALID, "wm_dense_i8: %d groups need offsets", G);
    WM_REQUIRE(N <= 1 << 20 && G <= 4096, WM_ERR_UNSUPPORTED, "wm_dense_i8: N=%d groups=%d is beyond 2^20 columns or 4096 groups", N, G);
    if (M == 0) return WM_OK;
    WM_REQUIRE(x && W && wscale && y, WM_ERR_INVALID, "wm_dense_i8: null pointer");
    const size_t need = wm_dense_i8_workspace_bytes(M, N, K);
    WM_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), WM_ERR_WORKSPACE, "wm_dense_i8: workspace of %zu bytes needed, %zu given", need,
               workspace_bytes);
    WM_REQUIRE(((uintptr_t)workspace & 15) == 0, WM_ERR_INVALID, "wm_dense_i8: workspace must be 16-byte aligned");
    hipStream_t st = (hipStream_t)stream;
    switch (dtype) {
    case WM_F32: return dense<float>(x, W, wscale, b, y, offsets, G, M, N, K, relu, workspace, st);
    case WM_BF16: return dense<bf16_t>(x, W, wscale, b, y, offsets, G, M, N, K, relu, workspace, st);
    default: return dense<f16_t>(x, W, wscale, b, y, offsets, G, M, N, K, relu, workspace, st);
    }
}
