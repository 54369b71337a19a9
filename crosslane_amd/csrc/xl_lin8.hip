// CDNA4 (gfx950) int8 product with a scale for each token and each output
// channel:
//
//   acc[t][r] = sum_k x[t][k] * w[r][k]                  exact, int32
//   out[t][r] = (float(acc) * x_scale[t]) * w_scale[r]
//   two matrices: g and u so, g = min(g, lim), u = clamp(u, -lim, lim) with a
//   limit, out = g / (1 + exp(-g)) * u
//
// v_mfma_i32_16x16x64_i8: lane l holds 16 consecutive k (16 (l / 16) ...) of row
// l % 16 of either operand, and of the result column l % 16, rows 4 (l / 16) + i.
// Tokens are the result's rows, channels its columns.
#include <hip/hip_ext.h>

#include "xl_act.hpp"

namespace xl::dev {
namespace {

typedef int v4i __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float swiglu1(float g, float u, float lim) {
    if (lim > 0.0f) {
        g = fminf(g, lim);
        u = fminf(fmaxf(u, -lim), lim);
    }
    return __fdiv_rn(g, 1.0f + expf(-g)) * u;
}

// 16 bytes of a row at k, those from K on zero.
__device__ __forceinline__ v4i row16(const int8_t* p, int k, int K, bool in) {
    v4i v{0, 0, 0, 0};
    if (in && k < K) {
        v = *reinterpret_cast<const v4i*>(p + k);
        if (k + 16 > K) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int left = K - k - 4 * i;   // bytes of this word inside the row
                v[i] &= left >= 4 ? -1 : left <= 0 ? 0 : (1 << (8 * left)) - 1;
            }
        }
    }
    return v;
}

// One wave: 16 tokens x 64 channels, straight from memory.
template <class OT, bool GATED>
__global__ __launch_bounds__(256) void lin8_simple_kernel(Lin8Args a) {
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    const int c = lane & 15, q = lane >> 4;
    const int64_t t0 = int64_t(blockIdx.y) * 16;
    const int64_t n0 = (int64_t(blockIdx.x) * 4 + wv) * 64;
    const int64_t t = t0 + c;
    const int8_t* xr = a.x + t * a.x_stride;
    v4i acc[4] = {}, acc2[4] = {};
    for (int k = 16 * q; k < a.K + 16 * q; k += 64) {
        const v4i xa = row16(xr, k, a.K, t < a.T);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int64_t n = n0 + 16 * j + c;
            acc[j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(xa, row16(a.w + n * a.w_stride, k, a.K, n < a.N), acc[j], 0, 0, 0);
            if constexpr (GATED)
                acc2[j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(xa, row16(a.up + n * a.w_stride, k, a.K, n < a.N), acc2[j], 0, 0, 0);
        }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int64_t n = n0 + 16 * j + c;
        if (n >= a.N) continue;
        const float ws = a.w_scale[n], us = GATED ? a.up_scale[n] : 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int64_t r = t0 + 4 * q + i;
            if (r >= a.T) continue;
            const float xs = a.x_scale[r];
            float y = float(acc[j][i]) * xs * ws;
            if constexpr (GATED) y = swiglu1(y, float(acc2[j][i]) * xs * us, a.lim);
            static_cast<OT*>(a.out)[r * a.out_stride + n] = rounded<OT>(y);
        }
    }
}

template <class OT>
void lin8_out(const Lin8Args& a, hipStream_t s, hipEvent_t stop) {
    const dim3 grid((a.N + 255) / 256, (a.T + 15) / 16);
    if (a.up) hipExtLaunchKernelGGL((lin8_simple_kernel<OT, true>), grid, dim3(256), 0, s, nullptr, stop, 0, a);
    else hipExtLaunchKernelGGL((lin8_simple_kernel<OT, false>), grid, dim3(256), 0, s, nullptr, stop, 0, a);
}

}  // namespace

hipError_t launch_lin8(const Lin8Args& a, int cus, hipStream_t s, hipEvent_t stop) {
    if (a.T < 1 || a.T > kLinMaxT || a.N < 1 || a.K < 1 || a.K > kLinMaxK || a.x_stride % 16 || a.w_stride % 16)
        return hipErrorInvalidValue;
    (void)cus;
    switch (a.out_type) {
    case kActF32: lin8_out<float>(a, s, stop); break;
    case kActF16: lin8_out<f16>(a, s, stop); break;
    case kActBF16: lin8_out<bf16>(a, s, stop); break;
    default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

}  // namespace xl::dev
