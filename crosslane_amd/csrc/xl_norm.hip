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
// norms and the quantization a call asks for: 8192 x 5120 in 16 bits at 4.3 TB/s, in
// float32 at 5.3, 2600 x 16000 in 16 bits at 3.6.
//
// Rows of more than 8192 values with a float32 among their types, and of more than 16384
// with any, are not there yet: nothing is loaded ahead, and four chunks of eight values a
// thread do not fit the 128 registers that sixteen waves leave each other, so 236 (all in 16
// bits) to 512 (all float32) bytes a thread go to scratch and back: 1300 x 32000 in 16 bits
// at 2.2 TB/s, in float32 at 1.4. Two chunks in float32 (up to 24 bytes): 1300 x 16000 at 3.1.
#include <hip/hip_ext.h>

#include <algorithm>

#include "xl_act.hpp"

namespace xl::dev {
namespace {

// A workgroup takes rows blockIdx.x, + gridDim.x, ...: with a row for each (few rows)
// or with several, the next row's loads on their way while this one is reduced and
// stored, and the vectors over the channels (post_w, pre_w, a gate for all) kept in
// registers, where one row for each workgroup would read as many bytes of them from L2
// as of the row itself. KEEP: registers allow that (rows of up to 8192 values, of 16384
// in 16 bits); else a row's loads follow the row before.
template <class T, class RT, int R, bool KEEP>
__global__ __launch_bounds__(1024, R == 1 ? 6 : 4) void block_norm_kernel(BlockNormArgs a) {
    __shared__ float red[2][3][16];
    const int NT = blockDim.x, D = a.D;
    int at[R];
#pragma unroll
    for (int j = 0; j < R; ++j) at[j] = 8 * (int(threadIdx.x) + j * NT);
    const bool one_gate = a.gate && a.gate_stride == 0;
    float post[KEEP ? R : 1][8], pre[KEEP ? R : 1][8];
    Eight<T> gate[R], y[R];
    Eight<RT> res[R];
    const auto fetch = [&](int64_t t) {
#pragma unroll
        for (int j = 0; j < R; ++j) {
            if (a.y) y[j] = eight(static_cast<const T*>(a.y) + t * a.y_stride + at[j], D - at[j]);
            if (a.res) res[j] = eight(static_cast<const RT*>(a.res) + t * a.res_stride + at[j], D - at[j]);
            if (a.gate && !one_gate) gate[j] = eight(static_cast<const T*>(a.gate) + t * a.gate_stride + at[j], D - at[j]);
        }
    };
    int64_t t = blockIdx.x;
    const auto of_channels = [&](int j) {
        if (a.post_w) load8(a.post_w + at[j], D - at[j], post[KEEP ? j : 0]);
        if (one_gate) gate[j] = eight(static_cast<const T*>(a.gate) + at[j], D - at[j]);
    };
    const auto before_next = [&](int j) { load8(a.pre_w + at[j], D - at[j], pre[KEEP ? j : 0]); };
    if (KEEP) {
        fetch(t);
#pragma unroll
        for (int j = 0; j < R; ++j) {
            of_channels(j);
            if (a.pre_w) before_next(j);
        }
    }
    for (int turn = 0; t < a.T; turn ^= 1) {
        if (!KEEP) fetch(t);
        float r[R][8];
        if (a.y) {
            float v[R][8], inv = 1.0f;
#pragma unroll
            for (int j = 0; j < R; ++j)
#pragma unroll
                for (int i = 0; i < 8; ++i) v[j][i] = float(y[j].v[i]);
            if (a.post_w) {
                float ss = 0.0f;
#pragma unroll
                for (int j = 0; j < R; ++j)
#pragma unroll
                    for (int i = 0; i < 8; ++i) ss = fmaf(v[j][i], v[j][i], ss);
                inv = 1.0f / sqrtf(group_join<false>(ss, red[turn][0]) / float(D) + a.eps);
            }
#pragma unroll
            for (int j = 0; j < R; ++j) {
                if (!KEEP) of_channels(j);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    float w = v[j][i];
                    if (a.post_w) w = w * inv * post[KEEP ? j : 0][i];
                    if (a.gate) w *= float(gate[j].v[i]);
                    r[j][i] = a.res ? fmaf(a.alpha, float(res[j].v[i]), w) : w;
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < R; ++j)
#pragma unroll
                for (int i = 0; i < 8; ++i) r[j][i] = a.alpha * float(res[j].v[i]);
        }
        const int64_t now = t;
        t += gridDim.x;
        if (KEEP && t < a.T) fetch(t);
        if (a.res_out) {
            RT* o = static_cast<RT*>(a.res_out) + now * a.res_out_stride;
#pragma unroll
            for (int j = 0; j < R; ++j) store8(o + at[j], D - at[j], r[j]);
        }
        if (!a.pre_w) continue;
        float ss = 0.0f;
#pragma unroll
        for (int j = 0; j < R; ++j)
#pragma unroll
            for (int i = 0; i < 8; ++i) ss = fmaf(r[j][i], r[j][i], ss);
        const float inv = 1.0f / sqrtf(group_join<false>(ss, red[turn][1]) / float(D) + a.eps);
#pragma unroll
        for (int j = 0; j < R; ++j) {
            if (!KEEP) before_next(j);
#pragma unroll
            for (int i = 0; i < 8; ++i) r[j][i] = r[j][i] * inv * pre[KEEP ? j : 0][i];
        }
        if (a.x) {
            T* o = static_cast<T*>(a.x) + now * a.x_stride;
#pragma unroll
            for (int j = 0; j < R; ++j) store8(o + at[j], D - at[j], r[j]);
        }
        if (!a.q) continue;
        float m = 0.0f;
#pragma unroll
        for (int j = 0; j < R; ++j) m = amax8(r[j], m);
        const float d = row_scale(group_join<true>(m, red[turn][2]), a.err);
        if (threadIdx.x == 0) a.q_scale[now] = d;
        int8_t* q = a.q + now * a.q_stride;
        const int end = (D + 15) & ~15;   // the quants' row ends with zeros to a multiple of 16
#pragma unroll
        for (int j = 0; j < R; ++j)
            if (at[j] < end) store_quants(q + at[j], r[j], d);
    }
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
hipError_t norm_types(const BlockNormArgs& a, int cus, hipStream_t s, hipEvent_t stop) {
    const int chunks = (a.D + 7) / 8;   // at most 4096
    constexpr bool NARROW = sizeof(T) + sizeof(RT) <= 4;   // two chunks for each thread fit its registers with all that is kept
    // Workgroups that a CU holds: their waves go round its four SIMDs, each workgroup from
    // the first one on, six to a SIMD with one chunk (80 registers), four with two (128).
    const auto held = [&](int per) {
        const int waves = row_threads(chunks, per) / 64, most = per == 1 ? 6 : 4;
        return waves < 4 ? most * 4 / waves : most / ((waves + 3) / 4);
    };
    // ... are launched, each with several rows: 8192 x 5120 bf16 in 79 us, with half as many
    // 109, with half as many again 120, with one for each row 106
    const auto go = [&](auto kernel, int per) {
        hipExtLaunchKernelGGL(kernel, dim3(std::min(a.T, cus * std::max(1, held(per)))), dim3(row_threads(chunks, per)), 0, s,
                              nullptr, stop, 0, a);
    };
    // two chunks where the CU then holds more rows: 2048 x 4096 to int8 in 19 us for 23, 1024 x 8192 in 20 for 27 (to
    // 16 bits 16 for 16 and 17 for 19)
    const bool two = NARROW && chunks > 256 && chunks <= 2048 && held(2) > held(1);
    if (chunks <= 1024 && !two) go(block_norm_kernel<T, RT, 1, true>, 1);
    else if (chunks <= 2048) go(block_norm_kernel<T, RT, 2, NARROW>, 2);
    else go(block_norm_kernel<T, RT, 4, false>, 4);
    return hipGetLastError();
}
template <class T>
hipError_t norm_type(const BlockNormArgs& a, int cus, hipStream_t s, hipEvent_t stop) {
    switch (a.res_type) {
    case kActF32: return norm_types<T, float>(a, cus, s, stop);
    case kActF16: return norm_types<T, f16>(a, cus, s, stop);
    case kActBF16: return norm_types<T, bf16>(a, cus, s, stop);
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

hipError_t launch_block_norm(const BlockNormArgs& a, int cus, hipStream_t s, hipEvent_t stop) {
    if (a.D < 1 || a.D > kNormMaxDim || a.T < 1 || (a.res_out && !a.y && !a.res) || (a.q && !a.pre_w) || (a.x && !a.pre_w))
        return hipErrorInvalidValue;
    switch (a.type) {
    case kActF32: return norm_type<float>(a, cus, s, stop);
    case kActF16: return norm_type<f16>(a, cus, s, stop);
    case kActBF16: return norm_type<bf16>(a, cus, s, stop);
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
