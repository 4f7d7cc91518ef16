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

constexpr int BLOCK = 256;

// bit j of the result: element e0 + j (j < 4) is dropped
__device__ __forceinline__ unsigned dropped4(uint64_t seed, uint64_t e0, unsigned sub, uint32_t upper, uint32_t lower)
{
    const uint64_t g = e0 >> 2;
    uint64_t w = hash64(seed, g);
    if (sub) w = (w >> (16 * sub)) | (hash64(seed, g + 1) << (64 - 16 * sub));
    unsigned drop = 0, tie = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const uint32_t d = (uint32_t)(w >> (16 * j)) & 0xFFFFu;
        drop |= (d < upper ? 1u : 0u) << j;
        tie |= (d == upper ? 1u : 0u) << j;
    }
    if (tie != 0 && lower != 0)
        for (int j = 0; j < 4; ++j)
            if (tie >> j & 1) {
                const uint64_t e = e0 + j;
                const uint64_t z = hash64(seed, hash64(seed, e >> 2));
                if (((uint32_t)(z >> (16 * (e & 3))) & 0xFFFFu) < lower) drop |= 1u << j;
            }
    return drop;
}

template <class T>
__global__ __launch_bounds__(BLOCK) void dropout_kernel(const T *__restrict__ x, const T *__restrict__ res, T *__restrict__ y,
                                                        long long n, uint64_t seed, uint64_t offset,
                                                        const long long *__restrict__ offset_dev, uint32_t upper,
                                                        uint32_t lower, float scale)
{
    const uint64_t base = offset + (offset_dev ? (uint64_t)*offset_dev : 0);
    const unsigned sub = (unsigned)(base & 3);
    for (long long i = ((long long)blockIdx.x * BLOCK + threadIdx.x) * 4; i < n; i += (long long)gridDim.x * BLOCK * 4) {
        const unsigned drop = dropped4(seed, base + (uint64_t)i, sub, upper, lower);
        for (int j = 0; j < 4 && i + j < n; ++j) {
            float v = drop >> j & 1 ? 0.0f : to_float(x[i + j]) * scale;
            if (res) v += to_float(res[i + j]);
            y[i + j] = from_float<T>(v);
        }
    }
}

template <class T>
int launch(const void *x, const void *res, void *y, long long n, uint64_t seed, uint64_t offset, const long long *offset_dev,
           uint64_t thr, hipStream_t st)
{
    const float scale = thr >> 32 ? 0.0f : (float)(0x1p32 / (0x1p32 - (double)thr));
    long long blocks = (n + 4 * BLOCK - 1) / (4 * BLOCK);
    if (blocks > 1 << 20) blocks = 1 << 20;
    hipLaunchKernelGGL(dropout_kernel<T>, dim3((unsigned)blocks), dim3(BLOCK), 0, st, (const T *)x, (const T *)res, (T *)y, n,
                       seed, offset, offset_dev, (uint32_t)(thr >> 16), (uint32_t)(thr & 0xFFFF), scale);
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
