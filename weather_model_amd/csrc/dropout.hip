// dropout.hip -- dropout whose mask is a function of (seed, element index) and is never stored.
//   forward   y[i]  = r[i] + (u(e) >= t ? x[i] / (1 - t 2^-32) : 0),   e = offset + i,  t = round(p 2^32)
//   backward  gx[i] =         u(e) >= t ? gy[i] / (1 - t 2^-32) : 0     (the same call without r)
// u(e) is a 32-bit draw: its upper half is bits 16 (e % 4) .. +15 of z = hash64(seed, e / 4), its lower half
// the same bits of hash64(seed, z).  The upper half decides all but one element in 65536, so one hash
// serves four elements and the second hash is only evaluated behind a branch that few waves take -- the
// probability keeps a resolution of 2^-32 at a quarter of a hash per element.
// A dropped element is an exact 0 (plus r) whatever x holds there, infinities and NaN included.
#include "common.h"
#include "hash64.h"
#include "half_types.h"

namespace {

constexpr int BLOCK = 256, UNROLL = 2;

// four draws of elements e0 .. e0 + 3, e0 = 4 g + sub: 16 bits each
__device__ __forceinline__ uint64_t draws4(uint64_t seed, uint64_t g, unsigned sub)
{
    uint64_t w = hash64(seed, g);
    if (sub) w = (w >> (16 * sub)) | (hash64(seed, g + 1) << (64 - 16 * sub));      // sub is the same for all lanes
    return w;
}

// drop[j] for elements e0 .. e0 + V - 1
template <int V>
__device__ __forceinline__ void draw(uint64_t seed, uint64_t e0, unsigned sub, uint32_t upper, uint32_t lower, bool (&drop)[V])
{
    bool tie = false;
#pragma unroll
    for (int h = 0; h < V / 4; ++h) {
        const uint64_t w = draws4(seed, (e0 >> 2) + h, sub);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t d = (uint32_t)(w >> (16 * j)) & 0xFFFFu;
            drop[4 * h + j] = d < upper;
            tie |= d == upper;
        }
    }
    if (lower != 0 && tie) {                     // one vector of 8 in 8192
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const uint64_t e = e0 + j, z = hash64(seed, e >> 2);
            if (((uint32_t)(z >> (16 * (e & 3))) & 0xFFFFu) == upper)
                drop[j] = ((uint32_t)(hash64(seed, z) >> (16 * (e & 3))) & 0xFFFFu) < lower;
        }
    }
}

// A thread takes UNROLL vectors of 16 bytes, BLOCK vectors apart: their loads go out before the first hash.
// Bound by HBM: 32768 x 2048 bf16 with a residual 76 us = 5.3 TB/s, without 43 us = 6.2 (a copy of 512 MiB 5.3); small calls by the launch.
template <class T, bool RES>
__global__ __launch_bounds__(BLOCK) void dropout_kernel(const T *x, const T *res, T *y,
                                                        long long n, uint64_t seed, uint64_t offset,
                                                        const long long *__restrict__ offset_dev, uint32_t upper,
                                                        uint32_t lower, float scale)
{
    constexpr int V = 16 / sizeof(T);
    typedef T vec __attribute__((ext_vector_type(V), aligned(sizeof(T))));
    const uint64_t base = offset + (offset_dev ? (uint64_t)*offset_dev : 0);
    const unsigned sub = (unsigned)(base & 3);
    constexpr long long SPAN = (long long)BLOCK * V * UNROLL;
    for (long long b = blockIdx.x * SPAN; b < n; b += gridDim.x * SPAN) {
        const long long i0 = b + threadIdx.x * V;
        if (b + SPAN <= n) {
            vec in[UNROLL], r[UNROLL];
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) {
                in[u] = *reinterpret_cast<const vec *>(x + i0 + u * BLOCK * V);
                if (RES) r[u] = *reinterpret_cast<const vec *>(res + i0 + u * BLOCK * V);
            }
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) {
                const long long i = i0 + u * BLOCK * V;
                bool drop[V];
                draw<V>(seed, base + (uint64_t)i, sub, upper, lower, drop);
                vec o;
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    float v = drop[j] ? 0.0f : to_float((T)in[u][j]) * scale;
                    if (RES) v += to_float((T)r[u][j]);
                    o[j] = from_float<T>(v);
                }
                *reinterpret_cast<vec *>(y + i) = o;
            }
        } else {
            for (long long i = i0; i < n; i += BLOCK * V) {
                bool drop[V];
                draw<V>(seed, base + (uint64_t)i, sub, upper, lower, drop);
#pragma unroll
                for (int j = 0; j < V; ++j)
                    if (i + j < n) {
                        float v = drop[j] ? 0.0f : to_float(x[i + j]) * scale;
                        if (RES) v += to_float(res[i + j]);
                        y[i + j] = from_float<T>(v);
                    }
            }
        }
    }
}

template <class T>
int launch(const void *x, const void *res, void *y, long long n, uint64_t seed, uint64_t offset, const long long *offset_dev,
           uint64_t thr, hipStream_t st)
{
    const float scale = thr >> 32 ? 0.0f : (float)(0x1p32 / (0x1p32 - (double)thr));
    constexpr long long SPAN = (long long)BLOCK * (16 / sizeof(T)) * UNROLL;
    long long blocks = (n + SPAN - 1) / SPAN;
    if (blocks > 1 << 20) blocks = 1 << 20;
    const uint32_t upper = (uint32_t)(thr >> 16), lower = (uint32_t)(thr & 0xFFFF);
    if (res)
        hipLaunchKernelGGL((dropout_kernel<T, true>), dim3((unsigned)blocks), dim3(BLOCK), 0, st, (const T *)x, (const T *)res, (T *)y, n, seed,
                           offset, offset_dev, upper, lower, scale);
    else
        hipLaunchKernelGGL((dropout_kernel<T, false>), dim3((unsigned)blocks), dim3(BLOCK), 0, st, (const T *)x, (const T *)nullptr, (T *)y, n,
                           seed, offset, offset_dev, upper, lower, scale);
    WM_LAUNCH_CHECK("dropout_kernel");
    return WM_OK;
}

}  // namespace

extern "C" int wm_dropout(const void *x, const void *residual, void *y, int64_t n, int dtype, double p, uint64_t seed,
                          uint64_t offset, const int64_t *offset_dev, void *stream)
{
    WM_REQUIRE(n >= 0, WM_ERR_INVALID, "wm_dropout: bad element count %lld", (long long)n);
    WM_REQUIRE(p >= 0.0 && p <= 1.0, WM_ERR_INVALID, "wm_dropout: p = %g is no probability", p);
    WM_REQUIRE(dtype == WM_F32 || dtype == WM_BF16 || dtype == WM_F16, WM_ERR_INVALID, "wm_dropout: bad dtype %d", dtype);
    if (n == 0) return WM_OK;
    WM_REQUIRE(x && y, WM_ERR_INVALID, "wm_dropout: null pointer");
    WM_REQUIRE(n <= ((int64_t)1 << 40), WM_ERR_UNSUPPORTED, "wm_dropout: more than 2^40 elements");
    WM_REQUIRE(wm_num_cus() > 0, WM_ERR_NO_DEVICE, "wm_dropout: no HIP device");
    const uint64_t thr = (uint64_t)__builtin_rint(p * 0x1p32);
    const long long *od = (const long long *)offset_dev;
    hipStream_t st = (hipStream_t)stream;
    switch (dtype) {
    case WM_F32: return launch<float>(x, residual, y, n, seed, offset, od, thr, st);
    case WM_BF16: return launch<bf16_t>(x, residual, y, n, seed, offset, od, thr, st);
    default: return launch<f16_t>(x, residual, y, n, seed, offset, od, thr, st);
    }
}
