// Activations of the calls that take more than float32 (xl_norm.hip,
// xl_score.hip, xl_lin8.hip): element types, chunks of eight values, and sums
// and maxima over a workgroup. gfx950 only.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

#include "xl_internal.hpp"

namespace xl::dev {

typedef _Float16 f16;
typedef __bf16 bf16;

// Eight consecutive values of a row, `n` of them in the row (the others 0). Rows start
// at any element: the loads are wide and unaligned (the hardware takes dword loads at
// any byte), so odd widths and strides go the same way as aligned ones.
template <class T>
struct Eight {
    T v[8];
};
template <class T>
__device__ __forceinline__ Eight<T> eight(const T* p, int n) {
    Eight<T> r;
    if (n >= 8) {
        __builtin_memcpy(&r, p, sizeof r);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) r.v[i] = i < n ? p[i] : T(0.0f);
    }
    return r;
}
template <class T>
__device__ __forceinline__ void load8(const T* p, int n, float (&v)[8]) {
    const Eight<T> r = eight(p, n);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = float(r.v[i]);
}
// The same to memory, each value rounded once (to nearest, ties to even).
template <class T>
__device__ __forceinline__ void store8(T* p, int n, const float (&v)[8]) {
    if (n >= 8) {
        T t[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) t[i] = T(v[i]);
        __builtin_memcpy(p, t, sizeof t);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) p[i] = T(v[i]);
    }
}

// A float32 product to an output type, in two roundings: left alone, a product and
// its conversion to f16 become one instruction that rounds once (v_fma_mixlo_f16),
// and f16 outputs then differ from the float32 ones rounded.
template <class T>
__device__ __forceinline__ T rounded(float v) {
    if constexpr (sizeof(T) == 2) asm("" : "+v"(v));
    return T(v);
}

// N (4 or 8) float32 products to memory, `n` of them in the row, in two roundings each (see `rounded`).
template <class T, int N>
__device__ __forceinline__ void store_rounded(T* p, int n, const float (&v)[N]) {
    if (n >= N) {
        T t[N];
#pragma unroll
        for (int i = 0; i < N; ++i) t[i] = rounded<T>(v[i]);
        __builtin_memcpy(p, t, sizeof t);
    } else {
#pragma unroll
        for (int i = 0; i < N - 1; ++i)
            if (i < n) p[i] = rounded<T>(v[i]);
    }
}

template <int CTRL, int MASK = 0xF>
__device__ __forceinline__ float dpp_or(float id, float v) {   // lanes that the pattern leaves out get `id`
    return __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(id), __float_as_int(v), CTRL, MASK, 0xF, false));
}
// Sum / maximum over the wave, in every lane; a fixed order.
template <bool MAX>
__device__ __forceinline__ float wave_join(float v) {
    const auto f = [](float a, float b) { return MAX ? fmaxf(a, b) : a + b; };
    v = f(v, dpp_or<0xB1>(0.0f, v));           // quad_perm 1,0,3,2
    v = f(v, dpp_or<0x4E>(0.0f, v));           // quad_perm 2,3,0,1
    v = f(v, dpp_or<0x141>(0.0f, v));          // row_half_mirror
    v = f(v, dpp_or<0x140>(0.0f, v));          // row_mirror
    v = f(v, dpp_or<0x142, 0xA>(0.0f, v));     // row_bcast:15 (maxima are of magnitudes: 0 is their identity)
    v = f(v, dpp_or<0x143, 0xC>(0.0f, v));     // row_bcast:31
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}
// The same over a workgroup of whole waves. `red`: 16 floats of LDS that no
// other call of the kernel uses (no barrier after the read).
template <bool MAX>
__device__ __forceinline__ float group_join(float v, float* red) {
    v = wave_join<MAX>(v);
    const int waves = int(blockDim.x) >> 6;
    if (waves == 1) return v;
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    float s = red[0];
    for (int i = 1; i < waves; ++i) s = MAX ? fmaxf(s, red[i]) : s + red[i];
    return s;
}

// Quantization of a row to int8 with one scale: d = max|x| / 127, q =
// round-half-even(x / d) in -127..127, separate IEEE roundings, so that equal
// rows give equal quants on any path. A row of zeros: d = 0, q = 0. A row with
// an infinity or a NaN: the device flag, q = 0 and d = NaN (its products are
// NaN, no finite wrong number).
//
// The quotient x / d of each value costs a dozen instructions; x times 1 / d rounds
// to the same whole number unless it lies within 2^-14 of a half: it is off by 127.5
// times 3 half steps at most (1 / d, the product, and the quotient's own rounding),
// 2.3e-5. So only groups of eight with such a value, and rows with a scale so small that
// 1 / d leaves the normal range, divide.
__device__ __forceinline__ uint32_t quant4(const float* v, float d) {
    uint32_t r = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float q = fminf(fmaxf(rintf(__fdiv_rn(v[i], d)), -127.0f), 127.0f);
        r |= (uint32_t(int(q)) & 0xffu) << (8 * i);
    }
    return d > 0.0f ? r : 0u;
}
// Eight quants at q[0..7]; those past the row (n..7) are zeros, written up to
// the next multiple of 16 bytes by whichever thread owns them.
__device__ __forceinline__ void store_quants(int8_t* q, const float (&v)[8], float d) {
    uint32_t o[2];
    const float inv = 1.0f / d;
    bool far = d >= 0x1p-100f;
    uint32_t n[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float t = v[i] * inv, m = t + 12582912.0f;   // 1.5 * 2^23: t rounded to a whole number, in the low bits
        n[i] = __float_as_uint(m);
        far = far && fabsf(t - (m - 12582912.0f)) < 0.5f - 0x1p-14f;
    }
    if (far) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
            o[i] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(n[4 * i + 3], n[4 * i + 2], 0x0c0c0400u),
                                         __builtin_amdgcn_perm(n[4 * i + 1], n[4 * i], 0x0c0c0400u), 0x05040100u);
    } else {
        o[0] = quant4(v, d);
        o[1] = quant4(v + 4, d);
    }
    __builtin_memcpy(q, o, 8);
}

// A row's scale from its largest magnitude (infinite where a value is not
// finite: the device flag, and a NaN).
__device__ __forceinline__ float row_scale(float amax, int* err) {
    if (amax <= 3.402823466e38f) return __fdiv_rn(amax, 127.0f);
    if (threadIdx.x == 0) atomicOr(err, kDevErrNonFinite);
    return __int_as_float(0x7fc00000);
}
__device__ __forceinline__ float amax8(const float (&v)[8], float m) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float a = fabsf(v[i]);
        m = a <= 3.402823466e38f ? fmaxf(m, a) : __int_as_float(0x7f800000);   // a NaN fails the comparison too
    }
    return m;
}

}  // namespace xl::dev
