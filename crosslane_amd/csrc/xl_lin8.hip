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

// Eight XCDs take workgroups in turn; tile `b` of `n` so that each XCD works on a
// run of consecutive tiles, and the tiles in groups of `gm` token tiles deep.
__device__ __forceinline__ void tile_of(int b, int tm, int tn, int& m, int& n) {
    const int all = tm * tn, x = b & 7, per = all >> 3, rest = all & 7;
    b = x * per + min(x, rest) + (b >> 3);
    constexpr int GM = 8;
    const int in_group = GM * tn, g = b / in_group, first = g * GM, deep = min(tm - first, GM);
    const int r = b - g * in_group;
    m = first + r % deep;
    n = r / deep;
}

// TT tokens x TC channels (of each matrix) per workgroup, WT x WC waves. Weights are
// the first operand: a lane's results are channels 4 q + i of one token. Row m of a
// wave's tile i is channel 4 NI (m / 4) + 4 i + m % 4 of the wave's, so that a lane has
// 4 NI consecutive channels and a token's are stored in runs of 16 NI.
template <class OT, bool GATED, int TT, int TC, int WT, int WC>
__global__ __launch_bounds__(64 * WT * WC, TT >= 256 ? 2 : 1) void lin8_tile_kernel(Lin8Args a, int tm, int tn) {
    constexpr int BK = 128, NT = 64 * WT * WC, M = GATED ? 2 : 1;
    constexpr int WTT = TT / WT, WTC = TC / WC;            // a wave's tokens and channels
    constexpr int NJ = WTT / 16, NI = WTC / 16;
    constexpr int LT = TT * BK / 16 / NT, LC = TC * BK / 16 / NT;   // 16-byte loads of a thread
    constexpr int RPL = NT / 8;                            // rows of one load of all threads
    __shared__ alignas(16) int8_t lds[2][(TT + M * TC) * BK];
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    const int c = lane & 15, q = lane >> 4;
    const int wt = wv / WC, wc = wv % WC;
    int bm, bn;
    tile_of(blockIdx.x, tm, tn, bm, bn);
    const int64_t t0 = int64_t(bm) * TT, n0 = int64_t(bn) * TC;
    const int8_t* xb = a.x + t0 * a.x_stride;
    const int8_t* wb = a.w + n0 * a.w_stride;
    const int8_t* ub = GATED ? a.up + n0 * a.w_stride : nullptr;
    const int row = tid >> 3, chunk = tid & 7;
    const int k16 = 16 * chunk;
    uint32_t offt[LT], offc[LC];
#pragma unroll
    for (int i = 0; i < LT; ++i)
        offt[i] = uint32_t(min(int64_t(row + i * RPL), int64_t(a.T) - 1 - t0)) * uint32_t(a.x_stride) + k16;
#pragma unroll
    for (int i = 0; i < LC; ++i) {
        const int r = row + i * RPL, in = r % WTC, m = in & 15;   // LDS row r: tile in / 16 of wave r / WTC, row m
        const int ch = r / WTC * WTC + 4 * NI * (m >> 2) + 4 * (in >> 4) + (m & 3);
        offc[i] = uint32_t(min(int64_t(ch), int64_t(a.N) - 1 - n0)) * uint32_t(a.w_stride) + k16;
    }
    // chunk p of row r lies at p ^ (r & 7): 16 rows of one chunk meet no bank twice
    const uint32_t put = uint32_t(row * BK + 16 * (chunk ^ (row & 7)));
    v4i gt[LT], gc[LC], gu[M == 2 ? LC : 1];
    const auto load = [&](int k) {
        if (k + BK <= a.K) {
#pragma unroll
            for (int i = 0; i < LT; ++i) gt[i] = *reinterpret_cast<const v4i*>(xb + k + offt[i]);
#pragma unroll
            for (int i = 0; i < LC; ++i) gc[i] = *reinterpret_cast<const v4i*>(wb + k + offc[i]);
            if constexpr (GATED)
#pragma unroll
                for (int i = 0; i < LC; ++i) gu[i] = *reinterpret_cast<const v4i*>(ub + k + offc[i]);
        } else {
#pragma unroll
            for (int i = 0; i < LT; ++i) gt[i] = row16(xb + offt[i] - k16, k + k16, a.K, true);
#pragma unroll
            for (int i = 0; i < LC; ++i) gc[i] = row16(wb + offc[i] - k16, k + k16, a.K, true);
            if constexpr (GATED)
#pragma unroll
                for (int i = 0; i < LC; ++i) gu[i] = row16(ub + offc[i] - k16, k + k16, a.K, true);
        }
    };
    const auto stage = [&](int8_t* b) {
#pragma unroll
        for (int i = 0; i < LT; ++i) *reinterpret_cast<v4i*>(b + put + i * RPL * BK) = gt[i];
#pragma unroll
        for (int i = 0; i < LC; ++i) *reinterpret_cast<v4i*>(b + TT * BK + put + i * RPL * BK) = gc[i];
        if constexpr (GATED)
#pragma unroll
            for (int i = 0; i < LC; ++i) *reinterpret_cast<v4i*>(b + (TT + TC) * BK + put + i * RPL * BK) = gu[i];
    };
    v4i acc[M][NI][NJ] = {};
    const uint32_t gett = uint32_t((wt * WTT + c) * BK), getc = uint32_t((TT + wc * WTC + c) * BK);
    const int steps = (a.K + BK - 1) / BK;
    load(0);
    stage(lds[0]);
    if (steps > 1) load(BK);
    __syncthreads();
    for (int s = 0; s < steps; ++s) {
        if (s + 1 < steps) stage(lds[(s + 1) & 1]);
        if (s + 2 < steps) load((s + 2) * BK);
        const int8_t* b = lds[s & 1];
#pragma unroll
        for (int h = 0; h < BK / 64; ++h) {
            const uint32_t at = 16 * ((4 * h + q) ^ (c & 7));
            v4i fw[M][NI];
#pragma unroll
            for (int m = 0; m < M; ++m)
#pragma unroll
                for (int i = 0; i < NI; ++i) fw[m][i] = *reinterpret_cast<const v4i*>(b + getc + (m * TC + 16 * i) * BK + at);
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                const v4i ft = *reinterpret_cast<const v4i*>(b + gett + 16 * j * BK + at);
#pragma unroll
                for (int m = 0; m < M; ++m)
#pragma unroll
                    for (int i = 0; i < NI; ++i)
                        acc[m][i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fw[m][i], ft, acc[m][i][j], 0, 0, 0);
            }
        }
        __syncthreads();
    }
    const int64_t n = n0 + wc * WTC + 4 * NI * q;
    const int left = int(min(int64_t(4 * NI), int64_t(a.N) - n));
    float ws[M][4 * NI];
#pragma unroll
    for (int e = 0; e < 4 * NI; ++e) {
        ws[0][e] = e < left ? a.w_scale[n + e] : 0.0f;
        if constexpr (GATED) ws[1][e] = e < left ? a.up_scale[n + e] : 0.0f;
    }
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
        const int64_t t = t0 + wt * WTT + 16 * j + c;
        if (t >= a.T) continue;
        const float xs = a.x_scale[t];
        OT* o = static_cast<OT*>(a.out) + t * a.out_stride + n;
#pragma unroll
        for (int i = 0; i < NI; i += 2) {
            float y[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                y[e] = float(acc[0][i + e / 4][j][e & 3]) * xs * ws[0][4 * i + e];
                if constexpr (GATED) y[e] = swiglu1(y[e], float(acc[1][i + e / 4][j][e & 3]) * xs * ws[1][4 * i + e], a.lim);
            }
            if (left > 4 * i) store8_rounded(o + 4 * i, left - 4 * i, y);
        }
    }
}

template <class OT, bool GATED, int TT, int TC, int WT, int WC>
void lin8_tiles(const Lin8Args& a, hipStream_t s, hipEvent_t stop) {
    const int tm = (a.T + TT - 1) / TT, tn = (a.N + TC - 1) / TC;
    hipExtLaunchKernelGGL((lin8_tile_kernel<OT, GATED, TT, TC, WT, WC>), dim3(tm * tn), dim3(64 * WT * WC), 0, s, nullptr, stop, 0, a, tm, tn);
}

template <class OT, bool GATED>
void lin8_out(const Lin8Args& a, hipStream_t s, hipEvent_t stop) {
    if (int64_t(a.T) * a.N >= 1024 * 1024 * 8) lin8_tiles<OT, GATED, 256, GATED ? 128 : 256, 2, 4>(a, s, stop);
    else lin8_tiles<OT, GATED, 128, GATED ? 64 : 128, 2, 2>(a, s, stop);
}

}  // namespace

hipError_t launch_lin8(const Lin8Args& a, int cus, hipStream_t s, hipEvent_t stop) {
    if (a.T < 1 || a.T > kLinMaxT || a.N < 1 || a.K < 1 || a.K > kLinMaxK || a.x_stride % 16 || a.w_stride % 16)
        return hipErrorInvalidValue;
    (void)cus;
    switch (a.out_type) {
    case kActF32: a.up ? lin8_out<float, true>(a, s, stop) : lin8_out<float, false>(a, s, stop); break;
    case kActF16: a.up ? lin8_out<f16, true>(a, s, stop) : lin8_out<f16, false>(a, s, stop); break;
    case kActBF16: a.up ? lin8_out<bf16, true>(a, s, stop) : lin8_out<bf16, false>(a, s, stop); break;
    default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

}  // namespace xl::dev
