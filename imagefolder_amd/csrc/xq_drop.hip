// xq_drop.hip — dropout whose mask is a function of (key, position) and is never stored (gfx950).
//
// y[i] = keep(i) ? x[i] * 65536 / (65536 - t) : 0   [+ residual[i]],   t = round(65536 p),   keep(i) = u16(i) >= t.
// u16(i): half i % 2 (low half first) of word (i % 8) / 2 of Philox4x32-10 (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy
// as 1, 2, 3", SC'11) at counter (i / 8 low, high, key[1] low, high) under the key (key[0] low, high).  The backward pass is the same map
// on the gradient, so nothing but the 16-byte key is kept between the two.
// Why 16 bits an element: one Philox call then serves the 8 elements of one 16-byte bf16 access.  32 bits an element would double the
// multiplies (20 of 32 x 32 -> 64 bits per call, a quarter of the VALU rate) and make them, not HBM, the bound.  HBM bounds it: 50.4 million elements bf16 + fp32
// residual -> fp32 105 us (4.8 TB/s), their gradient fp32 -> bf16 57 us (5.3 TB/s); the vector units are busy 18 and 32 % of the cycles.  p is rounded to a multiple of
// 2^-16; the factor uses the rounded one, so the expectation of y is x exactly.
#include "xq_common.hpp"
#include "xq_internal.hpp"
#include "xq_vec.hpp"
#include "../../include/xq_ops.h"
#include <algorithm>
#include <math.h>

namespace {

struct Words { uint32_t w[4]; };

__device__ __forceinline__ Words philox4x32_10(uint64_t block, uint64_t stream, uint64_t seed) {
    uint32_t a = (uint32_t)block, b = (uint32_t)(block >> 32), c = (uint32_t)stream, d = (uint32_t)(stream >> 32);
    uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const uint64_t p = (uint64_t)a * 0xD2511F53u, q = (uint64_t)c * 0xCD9E8D57u;
        a = (uint32_t)(q >> 32) ^ b ^ k0;
        b = (uint32_t)q;
        c = (uint32_t)(p >> 32) ^ d ^ k1;
        d = (uint32_t)p;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return Words{{a, b, c, d}};
}

// eight consecutive elements: one or two 16-byte accesses where VEC (every pointer 16-byte aligned), element by element otherwise
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T *p, long left, float (&v)[8]) {
    if (VEC && left >= 8) {
        load_vec<T, 8>(p, v);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = j < left ? to_f<T>(p[j]) : 0.0f;
    }
}

template <typename TX, typename TY, bool RES, bool VEC>
__global__ __launch_bounds__(256) void dropout_kernel(const TX *x, const TY *residual, long n, uint32_t threshold, float factor, const uint64_t *__restrict__ key,
                                                      TY *y) {                  // (no __restrict__: y may be x, a group's loads come before its stores)
    const uint64_t seed = key[0], stream = key[1];
    const long groups = (n + 7) / 8, step = (long)gridDim.x * 256;
    for (long g = (long)blockIdx.x * 256 + threadIdx.x; g < groups; g += step) {
        const long left = n - 8 * g;
        float v[8], r[8];
        load8<TX, VEC>(x + 8 * g, left, v);
        if (RES) load8<TY, VEC>(residual + 8 * g, left, r);
        const Words w = philox4x32_10((uint64_t)g, stream, seed);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint32_t u = (w.w[j >> 1] >> (16 * (j & 1))) & 0xffffu;
            const bool keep = u >= threshold;          // a dropped element is zero whatever x holds there (infinities, NaN)
            if (RES) v[j] = keep ? fmaf(v[j], factor, r[j]) : r[j];
            else v[j] = keep ? v[j] * factor : 0.0f;
        }
        if (VEC && left >= 8) {
            store_vec<TY, 8>(y + 8 * g, v);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (j < left) y[8 * g + j] = from_f<TY>(v[j]);
        }
    }
}

template <typename TX, typename TY>
void launch(const void *x, const void *residual, long n, uint32_t threshold, float factor, const void *key, void *y, hipStream_t s) {
    const bool vec = (((uintptr_t)x | (uintptr_t)residual | (uintptr_t)y) & 15) == 0;
    const long groups = (n + 7) / 8;
    const unsigned blocks = (unsigned)std::min<long>((groups + 255) / 256, (long)num_cus() * 16);
#define XQ_DROP(RES, VEC)                                                                                                                   \
    hipLaunchKernelGGL((dropout_kernel<TX, TY, RES, VEC>), dim3(blocks), dim3(256), 0, s, (const TX *)x, (const TY *)residual, n, threshold, \
                       factor, (const uint64_t *)key, (TY *)y)
    if (residual) { if (vec) XQ_DROP(true, true); else XQ_DROP(true, false); }
    else { if (vec) XQ_DROP(false, true); else XQ_DROP(false, false); }
#undef XQ_DROP
}

}  // namespace

extern "C" int xq_dropout(const void *x, int x_bf16, const void *residual, int64_t n, double p, const int64_t *key, void *y, int y_bf16,
                          xq_stream_t stream) {
    const char *fn = "xq_dropout";
    if (n < 0) return xq_set_error(XQ_EINVAL, "%s: negative size (%ld)", fn, (long)n);
    if (!(p >= 0.0 && p <= 1.0)) return xq_set_error(XQ_EINVAL, "%s: p must lie in [0, 1]", fn);
    if (n == 0) return XQ_OK;
    if (!x || !key || !y) return xq_set_error(XQ_EINVAL, "%s: null pointer", fn);
    if (((uintptr_t)key & 7) != 0) return xq_set_error(XQ_EINVAL, "%s: key must be 8-byte aligned", fn);
    const uint32_t t = (uint32_t)lrint(65536.0 * p);
    const float factor = t == 65536u ? 0.0f : (float)(65536.0 / (65536.0 - t));
    hipStream_t s = (hipStream_t)stream;
    if (x_bf16 && y_bf16) launch<bf16, bf16>(x, residual, n, t, factor, key, y, s);
    else if (x_bf16) launch<bf16, float>(x, residual, n, t, factor, key, y, s);
    else if (y_bf16) launch<float, bf16>(x, residual, n, t, factor, key, y, s);
    else launch<float, float>(x, residual, n, t, factor, key, y, s);
    return xq_check_launch(fn);
}
