// int8.hip -- Dense layers served in 8 bits: codes with one scale per row (token) and per channel.
//   quantise  s_m = max_k |x[m][k]| / 127 (float32), q[m][k] = round(x[m][k] / s_m) to even, within +-127
//   product   y[m][n] = act((sum_k q[m][k] w[n][k]) s_m t_n + b[n]),  w (N, K) codes and t (N) scales of the weights
// The integer sum is exact (K <= 2^17 keeps it within 32 bits, -128 among the codes included); it is rounded
// to float32 once and scaled there.  A row of zeros has s = 0 and codes 0; a row that holds an infinity or a
// NaN has s = NaN and codes 0, so that all its outputs are NaN.
#include "few_rows.h"

namespace {

using namespace tile;

constexpr int THREADS = 256;                 // of the kernels without tiles

// One workgroup a row.  Codes go to q with row stride ldq >= K, zeros behind K.
template <class E>
__global__ __launch_bounds__(THREADS) void quantize_rows_kernel(const E *__restrict__ x, int K, int8_t *__restrict__ q, long long ldq,
                                                                float *__restrict__ scale)
{
    __shared__ float part[4];
    const long long m = blockIdx.x;
    const E *row = x + m * K;
    float top = 0.0f;
    bool bad = false;
    for (int k = threadIdx.x; k < K; k += THREADS) {
        const float a = fabsf(to_float(row[k]));
        bad |= !(a <= 3.4028235e38f);
        top = fmaxf(top, a);
    }
    if (bad) top = __builtin_nanf("");
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const float t = __shfl_xor(top, o, 64);
        top = top != top || t != t ? __builtin_nanf("") : fmaxf(top, t);
    }
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = top;
    __syncthreads();
    float s = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; ++w) s = part[w] != part[w] || s != s ? __builtin_nanf("") : fmaxf(s, part[w]);
    s = s / 127.0f;
    for (int k = threadIdx.x; k < ldq; k += THREADS) {
        float c = 0.0f;
        if (k < K && s > 0.0f) c = fminf(fmaxf(rintf(to_float(row[k]) / s), -127.0f), 127.0f);
        q[m * ldq + k] = (int8_t)c;
    }
    if (threadIdx.x == 0) scale[m] = s;
}

template <class E, class S>
__global__ __launch_bounds__(S::THREADS) void dense_i8_kernel(const int8_t *__restrict__ q, long long ldq, const float *__restrict__ qscale,
                                                           const int8_t *__restrict__ W, const float *__restrict__ wscale,
                                                           const float *__restrict__ bias, E *__restrict__ y,
                                                           const long long *__restrict__ offsets, int G, int M, int N, int K, int relu, int band)
{
    constexpr int BM = S::BM, BN = S::BN, THREADS = S::THREADS;
    __shared__ __attribute__((aligned(16))) char lds[S::LDS];
    int rt, ct;
    if (!tile_of_block(blockIdx.x, row_tiles(offsets, G, M, BM), (N + BN - 1) / BN, band, rt, ct)) return;
    const Segment s = row_tile(offsets, G, M, BM, rt);
    const int n0 = min(ct * BN, max(0, N - BN)), cols = min(BN, N);         // the last tile moves back over its neighbour
    if (s.g < 0 || s.g >= G) {                       // rows of no expert: zeros
        for (int e = threadIdx.x; e < s.rows * cols; e += THREADS) y[(long long)(s.row0 + e / cols) * N + n0 + e % cols] = (E)0.0f;
        return;
    }
    Contiguous<I8, BN, THREADS> a;
    Contiguous<I8, BM, THREADS> b;
    a.init(W + ((long long)s.g * N + n0) * K, K, cols, K, W + (long long)G * N * K);
    b.init(q + s.row0 * ldq, ldq, s.rows, K, q + M * ldq);
    constexpr int MI = S::MI, NI = S::NI;
    typename S::Acc acc = {};
    product<S>(a, b, K, lds, acc);
    const int ni0 = S::col(), mi0 = S::row();
#pragma unroll
    for (int m = 0; m < MI; ++m) {
        const int r = mi0 + 16 * m;
        if (r >= s.rows) continue;
        const long long row = (long long)(s.row0 + r) * N + n0;
        const float qs = qscale[s.row0 + r];
#pragma unroll
        for (int n = 0; n < NI; ++n) {
            const int i = ni0 + 16 * n;
            if (i >= cols) continue;
            const int have = min(4, cols - i);
            const long long c = (long long)s.g * N + n0 + i;
            f32x4 v;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int kk = min(k, have - 1);
                v[k] = (float)acc[m][n][k] * qs * wscale[c + kk] + (bias ? bias[c + kk] : 0.0f);
                if (relu) v[k] = relu_of(v[k]);
            }
            if (have == 4) store4(y + row + i, v);
            else
                for (int k = 0; k < have; ++k) y[row + i + k] = from_float<E>(v[k]);
        }
    }
}

// ---- few rows: one read of the weights (few_rows.h)
template <class E>
__global__ __launch_bounds__(few::THREADS) void dense_i8_few_kernel(const int8_t *__restrict__ q, long long ldq, const float *__restrict__ qscale,
                                                                    const int8_t *__restrict__ W, const float *__restrict__ wscale,
                                                                    const float *__restrict__ bias, E *__restrict__ y,
                                                                    const long long *__restrict__ offsets, int G, int M, int N, int K, int relu)
{
    __shared__ i32x4 part[few::WAVES][64];
    const int g = blockIdx.y, n0 = blockIdx.x * 16, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int row0 = 0, rows = M;
    if (g == G) {                                    // rows of no expert: zeros
        int end;
        group_rows(offsets, G, M, 0, row0, rows);
        group_rows(offsets, G, M, G - 1, end, rows);
        end += rows;
        const int cols = min(16, N - n0);
        for (int e = threadIdx.x; e < (row0 + M - end) * cols; e += few::THREADS) {
            const int r = e / cols;
            y[(long long)(r < row0 ? r : r - row0 + end) * N + n0 + e % cols] = (E)0.0f;
        }
        return;
    }
    if (offsets) group_rows(offsets, G, M, g, row0, rows);
    const int8_t *wrow = W + ((long long)g * N + min(n0 + (lane & 15), N - 1)) * K;
    for (int r0 = 0; r0 < rows; r0 += 16) {
        const int r = min(r0 + (lane & 15), rows - 1);
        const i32x4 acc = few::dot<I8>(wrow, W + (long long)G * N * K, q + (row0 + r) * ldq, q + M * ldq, K);
        if (wave > 0) part[wave][lane] = acc;
        __syncthreads();
        if (wave == 0) {
            i32x4 s = acc;
#pragma unroll
            for (int w = 1; w < few::WAVES; ++w) s += part[w][lane];
            const int n = n0 + 4 * (lane >> 4), have = min(4, N - n);
            if (r0 + (lane & 15) < rows && have > 0) {
                E *at = y + (long long)(row0 + r) * N + n;
                const float qs = qscale[row0 + r];
                const long long c = (long long)g * N + n;
                f32x4 v;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int kk = min(k, have - 1);
                    v[k] = (float)s[k] * qs * wscale[c + kk] + (bias ? bias[c + kk] : 0.0f);
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

template <class E> int quantize(const void *x, int M, int K, int8_t *q, long long ldq, float *scale, hipStream_t st)
{
    hipLaunchKernelGGL(quantize_rows_kernel<E>, dim3(M), dim3(THREADS), 0, st, (const E *)x, K, q, ldq, scale);
    WM_LAUNCH_CHECK("quantize_rows_kernel");
    return WM_OK;
}

template <class E, class S>
int dense_tiles(const int8_t *q, long long ldq, const float *scale, const int8_t *W, const float *wscale, const float *b, void *y,
                const int64_t *offsets, int G, int M, int N, int K, int relu, hipStream_t st)
{
    const long long blocks = row_tiles_most(G, M, S::BM) * ((N + S::BN - 1) / S::BN);
    WM_REQUIRE(blocks <= (1ll << 32) / 512 - 1, WM_ERR_UNSUPPORTED, "wm_dense_i8: %lld tiles are too many for one launch", blocks);
    hipLaunchKernelGGL((dense_i8_kernel<E, S>), dim3((unsigned)blocks), dim3(S::THREADS), 0, st, q, ldq, scale, W, wscale, b, (E *)y,
                       (const long long *)offsets, G, M, N, K, relu, 8);
    WM_LAUNCH_CHECK("dense_i8_kernel");
    return WM_OK;
}

template <class E>
int dense(const void *x, const int8_t *W, const float *wscale, const float *b, void *y, const int64_t *offsets, int G, int M, int N, int K, int relu,
          void *workspace, hipStream_t st)
{
    float *scale = (float *)workspace;
    int8_t *q = (int8_t *)workspace + wm_align_up((size_t)M * sizeof(float), 256);
    const long long ldq = (long long)padded(K);
    if (int rc = quantize<E>(x, M, K, q, ldq, scale, st)) return rc;
    if ((M <= 64 || M / G <= 8) && G < 65535) {
        hipLaunchKernelGGL(dense_i8_few_kernel<E>, dim3((N + 15) / 16, offsets ? G + 1 : 1), dim3(few::THREADS), 0, st, q, ldq, scale, W, wscale, b,
                           (E *)y, (const long long *)offsets, G, M, N, K, relu);
        WM_LAUNCH_CHECK("dense_i8_few_kernel");
        return WM_OK;
    }
    if (M / G >= 512 && N >= 512) return dense_tiles<E, Shape<I8, 256, 256, 2, 4>>(q, ldq, scale, W, wscale, b, y, offsets, G, M, N, K, relu, st);
    return dense_tiles<E, Shape<I8, 128, 128, 2, 2>>(q, ldq, scale, W, wscale, b, y, offsets, G, M, N, K, relu, st);
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

extern "C" size_t wm_dense_i8_workspace_bytes(int M, int K)
{
    if (M <= 0 || K <= 0) return 0;
    return wm_align_up((size_t)M * sizeof(float), 256) + (size_t)M * padded(K);
}

extern "C" int wm_dense_i8(const void *x, const int8_t *W, const float *wscale, const float *b, void *y, const int64_t *offsets, int G, int M,
                           int N, int K, int dtype, int relu, void *workspace, size_t workspace_bytes, void *stream)
{
    if (int rc = check("wm_dense_i8", M, K, dtype)) return rc;
    WM_REQUIRE(N > 0 && G > 0, WM_ERR_INVALID, "wm_dense_i8: bad sizes N=%d groups=%d", N, G);
    WM_REQUIRE(offsets || G == 1, WM_ERR_INVALID, "wm_dense_i8: %d groups need offsets", G);
    WM_REQUIRE(N <= 1 << 20 && G <= 1 << 16, WM_ERR_UNSUPPORTED, "wm_dense_i8: N=%d groups=%d is beyond 2^20 columns or 2^16 groups", N, G);
    if (M == 0) return WM_OK;
    WM_REQUIRE(x && W && wscale && y, WM_ERR_INVALID, "wm_dense_i8: null pointer");
    const size_t need = wm_dense_i8_workspace_bytes(M, K);
    WM_REQUIRE(workspace && workspace_bytes >= need, WM_ERR_WORKSPACE, "wm_dense_i8: workspace of %zu bytes needed, %zu given", need,
               workspace_bytes);
    WM_REQUIRE(((uintptr_t)workspace & 15) == 0, WM_ERR_INVALID, "wm_dense_i8: workspace must be 16-byte aligned");
    hipStream_t st = (hipStream_t)stream;
    switch (dtype) {
    case WM_F32: return dense<float>(x, W, wscale, b, y, offsets, G, M, N, K, relu, workspace, st);
    case WM_BF16: return dense<bf16_t>(x, W, wscale, b, y, offsets, G, M, N, K, relu, workspace, st);
    default: return dense<f16_t>(x, W, wscale, b, y, offsets, G, M, N, K, relu, workspace, st);
    }
}
