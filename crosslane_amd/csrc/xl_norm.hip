// CDNA4 (gfx950) kernels of what lies between two blocks with an ordinary
// residual stream, and of the row quantizer that feeds the int8 product.
//
//   a = y                                                   the block's output
//   a = a * 1 / sqrt(mean(a^2) + eps) * post_w              with post_w
//   r = alpha * res + gate * a                              (no gate: 1; no res: 0)
//   x = r * 1 / sqrt(mean(r^2) + eps) * pre_w               with pre_w
//   q, d = x quantized to int8, a scale for the row         with q
//
// All in float32, x from the unrounded r, one rounding at each store.
//
// Bound by memory: one workgroup per row holds the row in registers, so y, res
// and gate are read once and r, x or q written once, however many of the two
// norms and the quantization a call asks for.
#include <hip/hip_ext.h>

#include <algorithm>

#include "xl_act.hpp"

namespace xl::dev {
namespace {

template <class T, class RT, int R>
__global__ __launch_bounds__(1024) void block_norm_kernel(BlockNormArgs a) {
    __shared__ float red[4][16];
    const int64_t t = blockIdx.x;
    const int NT = blockDim.x, D = a.D;
    float v[R][8], r[R][8];
    int at[R];
#pragma unroll
    for (int j = 0; j < R; ++j) at[j] = 8 * (int(threadIdx.x) + j * NT);
    const T* y = static_cast<const T*>(a.y) + t * a.y_stride;
    const RT* res = static_cast<const RT*>(a.res) + t * a.res_stride;
    const T* gate = static_cast<const T*>(a.gate) + t * a.gate_stride;
#pragma unroll
    for (int j = 0; j < R; ++j) {
        if (a.res) load8(res + at[j], D - at[j], r[j]);
        else
            for (int i = 0; i < 8; ++i) r[j][i] = 0.0f;
        if (a.y) load8(y + at[j], D - at[j], v[j]);
    }
    if (a.y) {
        float inv = 1.0f;
        if (a.post_w) {
            float ss = 0.0f;
#pragma unroll
            for (int j = 0; j < R; ++j)
#pragma unroll
                for (int i = 0; i < 8; ++i) ss = fmaf(v[j][i], v[j][i], ss);
            inv = 1.0f / sqrtf(group_join<false>(ss, red[0]) / float(D) + a.eps);
        }
#pragma unroll
        for (int j = 0; j < R; ++j) {
            float w[8];
            if (a.post_w) {
                load8(a.post_w + at[j], D - at[j], w);
#pragma unroll
                for (int i = 0; i < 8; ++i) v[j][i] = v[j][i] * inv * w[i];
            }
            if (a.gate) {
                load8(gate + at[j], D - at[j], w);
#pragma unroll
                for (int i = 0; i < 8; ++i) v[j][i] *= w[i];
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) r[j][i] = fmaf(a.alpha, r[j][i], v[j][i]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < R; ++j)
#pragma unroll
            for (int i = 0; i < 8; ++i) r[j][i] *= a.alpha;
    }
    if (a.res_out) {
        RT* o = static_cast<RT*>(a.res_out) + t * a.res_out_stride;
#pragma unroll
        for (int j = 0; j < R; ++j) store8(o + at[j], D - at[j], r[j]);
    }
    if (!a.pre_w) return;
    float ss = 0.0f;
#pragma unroll
    for (int j = 0; j < R; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) ss = fmaf(r[j][i], r[j][i], ss);
    const float inv = 1.0f / sqrtf(group_join<false>(ss, red[1]) / float(D) + a.eps);
#pragma unroll
    for (int j = 0; j < R; ++j) {
        float w[8];
        load8(a.pre_w + at[j], D - at[j], w);
#pragma unroll
        for (int i = 0; i < 8; ++i) r[j][i] = r[j][i] * inv * w[i];
    }
    if (a.x) {
        T* o = static_cast<T*>(a.x) + t * a.x_stride;
#pragma unroll
        for (int j = 0; j < R; ++j) store8(o + at[j], D - at[j], r[j]);
    }
    if (!a.q) return;
    float m = 0.0f;
#pragma unroll
    for (int j = 0; j < R; ++j) m = amax8(r[j], m);
    const float d = row_scale(group_join<true>(m, red[2]), a.err);
    if (threadIdx.x == 0) a.q_scale[t] = d;
    int8_t* q = a.q + t * a.q_stride;
    const int end = (D + 15) & ~15;   // the quants' row ends with zeros to a multiple of 16
#pragma unroll
    for (int j = 0; j < R; ++j)
        if (at[j] < end) store_quants(q + at[j], r[j], d);
}

// Rows to int8 with a scale each. R > 0: the row in registers; R == 0: rows of
// any length, read twice (the second time from a cache).
template <class T, int R>
__global__ __launch_bounds__(1024) void quant_rows_kernel(const T* __restrict__ x, int64_t x_stride, int K,
                                                          int8_t* __restrict__ q, int64_t q_stride,
                                                          float* __restrict__ scale, int* err) {
    __shared__ float red[16];
    const int64_t t = blockIdx.x;
    const int NT = blockDim.x;
    const int end = (K + 15) & ~15;
    x += t * x_stride;
    q += t * q_stride;
    float m = 0.0f;
    if constexpr (R > 0) {
        float v[R][8];
#pragma unroll
        for (int j = 0; j < R; ++j) {
            const int at = 8 * (int(threadIdx.x) + j * NT);
            load8(x + at, K - at, v[j]);
        }
#pragma unroll
        for (int j = 0; j < R; ++j) m = amax8(v[j], m);
        const float d = row_scale(group_join<true>(m, red), err);
        if (threadIdx.x == 0) scale[t] = d;
#pragma unroll
        for (int j = 0; j < R; ++j) {
            const int at = 8 * (int(threadIdx.x) + j * NT);
            if (at < end) store_quants(q + at, v[j], d);
        }
    } else {
        float v[8];
        for (int at = 8 * int(threadIdx.x); at < K; at += 8 * NT) {
            load8(x + at, K - at, v);
            m = amax8(v, m);
        }
        const float d = row_scale(group_join<true>(m, red), err);
        if (threadIdx.x == 0) scale[t] = d;
        for (int at = 8 * int(threadIdx.x); at < end; at += 8 * NT) {
            load8(x + at, K - at, v);
            store_quants(q + at, v, d);
        }
    }
}

// Threads for rows of n chunks of eight values, `per` chunks each.
int row_threads(int n, int per) { return std::min(1024, ((n + per - 1) / per + 63) / 64 * 64); }

template <class T, class RT>
hipError_t norm_types(const BlockNormArgs& a, hipStream_t s, hipEvent_t stop) {
    const int chunks = (a.D + 7) / 8;   // at most 4096
    const auto go = [&](auto kernel, int per) {
        hipExtLaunchKernelGGL(kernel, dim3(a.T), dim3(row_threads(chunks, per)), 0, s, nullptr, stop, 0, a);
    };
    if (chunks <= 1024) go(block_norm_kernel<T, RT, 1>, 1);
    else if (chunks <= 2048) go(block_norm_kernel<T, RT, 2>, 2);
    else go(block_norm_kernel<T, RT, 4>, 4);
    return hipGetLastError();
}
template <class T>
hipError_t norm_type(const BlockNormArgs& a, hipStream_t s, hipEvent_t stop) {
    switch (a.res_type) {
    case kActF32: return norm_types<T, float>(a, s, stop);
    case kActF16: return norm_types<T, f16>(a, s, stop);
    case kActBF16: return norm_types<T, bf16>(a, s, stop);
    default: return hipErrorInvalidValue;
    }
}
template <class T>
hipError_t quant_type(const void* x, int64_t x_stride, int T_, int K, int8_t* q, int64_t q_stride, float* scale, int* err,
                      hipStream_t s, hipEvent_t stop) {
    const int chunks = (K + 7) / 8;
    const auto go = [&](auto kernel, int per) {
        hipExtLaunchKernelGGL(kernel, dim3(T_), dim3(row_threads(chunks, per)), 0, s, nullptr, stop, 0,
                              static_cast<const T*>(x), x_stride, K, q, q_stride, scale, err);
    };
    if (chunks <= 1024) go(quant_rows_kernel<T, 1>, 1);
    else if (chunks <= 4096) go(quant_rows_kernel<T, 4>, 4);
    else go(quant_rows_kernel<T, 0>, 8);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_block_norm(const BlockNormArgs& a, hipStream_t s, hipEvent_t stop) {
    if (a.D < 1 || a.D > kNormMaxDim || a.T < 1 || (a.res_out && !a.y && !a.res) || (a.q && !a.pre_w) || (a.x && !a.pre_w))
        return hipErrorInvalidValue;
    switch (a.type) {
    case kActF32: return norm_type<float>(a, s, stop);
    case kActF16: return norm_type<f16>(a, s, stop);
    case kActBF16: return norm_type<bf16>(a, s, stop);
    default: return hipErrorInvalidValue;
    }
}

hipError_t launch_quant_rows(const void* x, int type, int64_t x_stride, int T, int K, int8_t* q, int64_t q_stride,
                             float* scale, int* err, hipStream_t s, hipEvent_t stop) {
    if (T < 1 || K < 1) return hipErrorInvalidValue;
    switch (type) {
    case kActF32: return quant_type<float>(x, x_stride, T, K, q, q_stride, scale, err, s, stop);
    case kActF16: return quant_type<f16>(x, x_stride, T, K, q, q_stride, scale, err, s, stop);
    case kActBF16: return quant_type<bf16>(x, x_stride, T, K, q, q_stride, scale, err, s, stop);
    default: return hipErrorInvalidValue;
    }
}

}  // namespace xl::dev
