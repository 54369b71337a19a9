// CDNA4 (gfx950) router over softmax or sigmoid scores:
//
//   s_e = exp(l_e - max l) / sum exp(l - max l)     or     1 / (1 + exp(-l_e))
//   key_e = s_e + bias_e
//   groups of n / G consecutive experts, each worth the sum of its one or two
//   largest keys: the top_groups of them by value stay
//   the k largest keys of the groups that stay: weight s_e, divided by the sum of
//   the picked (+ 1e-20) with renorm, times scale
//
// Ties go to the lower index. An expert whose logit is -inf is masked: s = 0 and
// key = -1e300, so it comes after every other of its group and keeps the row's
// picks whole (with weight 0) where fewer than k are left.
//
// Scores and keys are doubles: picks are whole numbers, and two of 256 sigmoid
// scores lie closer than float32 resolves in a few of ten thousand tokens. The
// vector units do a double operation at the rate of a float one.
#include <hip/hip_ext.h>

#include "xl_act.hpp"
#include "xl_route.hpp"

namespace xl::dev {
namespace {

constexpr double kMaskedKey = -1e300;

// Keys as unsigned integers that order as the doubles do; 0 for what is out.
__device__ __forceinline__ uint64_t ordered64(double d) {
    const uint64_t u = __double_as_longlong(d);
    return (u >> 63) ? ~u : (u | 0x8000000000000000ull);
}
__device__ __forceinline__ double unordered64(uint64_t u) {
    return __longlong_as_double(int64_t((u >> 63) ? (u ^ 0x8000000000000000ull) : ~u));
}
template <int CTRL, int MASK = 0xF>
__device__ __forceinline__ uint64_t dpp64(uint64_t v) {   // 0 in lanes that the pattern leaves out
    const uint32_t lo = uint32_t(__builtin_amdgcn_update_dpp(0, int(uint32_t(v)), CTRL, MASK, 0xF, false));
    const uint32_t hi = uint32_t(__builtin_amdgcn_update_dpp(0, int(uint32_t(v >> 32)), CTRL, MASK, 0xF, false));
    return uint64_t(lo) | (uint64_t(hi) << 32);
}
__device__ __forceinline__ uint64_t readlane64(uint64_t v, int lane) {
    const uint32_t lo = uint32_t(__builtin_amdgcn_readlane(int(uint32_t(v)), lane));
    const uint32_t hi = uint32_t(__builtin_amdgcn_readlane(int(uint32_t(v >> 32)), lane));
    return uint64_t(lo) | (uint64_t(hi) << 32);
}
template <class F>
__device__ __forceinline__ uint64_t wave_fold64(uint64_t v, F f) {   // identity 0
    v = f(v, dpp64<0xB1>(v));
    v = f(v, dpp64<0x4E>(v));
    v = f(v, dpp64<0x141>(v));
    v = f(v, dpp64<0x140>(v));
    v = f(v, dpp64<0x142, 0xA>(v));
    v = f(v, dpp64<0x143, 0xC>(v));
    return readlane64(v, 63);
}
__device__ __forceinline__ uint64_t wave_max64(uint64_t v) {
    return wave_fold64(v, [](uint64_t a, uint64_t b) { return a > b ? a : b; });
}
__device__ __forceinline__ double wave_sum64(double v) {
    return __longlong_as_double(int64_t(wave_fold64(uint64_t(__double_as_longlong(v)), [](uint64_t a, uint64_t b) {
        return uint64_t(__double_as_longlong(__longlong_as_double(int64_t(a)) + __longlong_as_double(int64_t(b))));
    })));
}

// One wave per token, expert lane + 64 j in slot j of each lane. Group values
// through LDS: lane g reads group g's keys.
template <class T, int NPL>
__global__ __launch_bounds__(256) void score_route_kernel(ScoreArgs a) {
    constexpr int WAVES = 4;
    __shared__ uint64_t keys[WAVES][NPL * 64];
    __shared__ double values[WAVES][NPL * 64];
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    const int64_t t = int64_t(blockIdx.x) * WAVES + wv;
    const bool here = t < a.T;   // every wave reaches the barriers
    const T* lg = static_cast<const T*>(a.logits) + (here ? t : 0) * a.stride;
    float l[NPL];
    float top = -__int_as_float(0x7f800000);
    bool bad = false;
#pragma unroll
    for (int j = 0; j < NPL; ++j) {
        const int e = lane + 64 * j;
        l[j] = e < a.n ? float(lg[e]) : -__int_as_float(0x7f800000);
        bad |= !(l[j] <= 3.402823466e38f);
        top = fmaxf(top, l[j]);
    }
    // the largest logit, by integers that order as floats do
    const uint32_t ot = wave_ext<true>(ordered(top));
    top = __uint_as_float((ot & 0x80000000u) ? (ot ^ 0x80000000u) : ~ot);
    const double dtop = top >= -3.402823466e38f ? double(top) : 0.0;
    double p[NPL], total = 0.0;
#pragma unroll
    for (int j = 0; j < NPL; ++j) {
        const double x = double(l[j]);
        const bool on = l[j] >= -3.402823466e38f;
        p[j] = !on ? 0.0 : a.sigmoid ? 1.0 / (1.0 + exp(-x)) : exp(x - dtop);
        total += p[j];
    }
    double denom = 1.0;
    if (!a.sigmoid) {
        denom = wave_sum64(total);
        denom = denom > 0.0 ? denom : 1.0;
    }
    uint64_t key[NPL];
#pragma unroll
    for (int j = 0; j < NPL; ++j) {
        const int e = lane + 64 * j;
        const float b = a.bias && e < a.n ? a.bias[e] : 0.0f;
        const bool on = l[j] >= -3.402823466e38f;
        bad |= !(fabsf(b) <= 3.402823466e38f);
        const double s = a.sigmoid ? p[j] : p[j] / denom;
        key[j] = e < a.n ? ordered64(on ? s + double(b) : kMaskedKey) : 0;
    }
    if (__any(bad) && here && lane == 0) atomicOr(a.err, kDevErrNonFinite);
    if (a.groups > 1) {
        const int size = a.n / a.groups;
#pragma unroll
        for (int j = 0; j < NPL; ++j) keys[wv][lane + 64 * j] = key[j];
        __syncthreads();
        for (int g = lane; g < a.groups; g += 64) {
            uint64_t m1 = 0, m2 = 0;
            for (int i = 0; i < size; ++i) {
                const uint64_t v = keys[wv][g * size + i];
                if (v > m1) { m2 = m1; m1 = v; }
                else if (v > m2) m2 = v;
            }
            values[wv][g] = unordered64(m1) + (a.group_keys == 2 ? unordered64(m2) : 0.0);
        }
        __syncthreads();
        // a group stays if fewer than top_groups are ahead of it
#pragma unroll
        for (int j = 0; j < NPL; ++j) {
            const int g = (lane + 64 * j) / size;
            if (lane + 64 * j >= a.n) continue;
            const double mine = values[wv][g];
            int ahead = 0;
            for (int i = 0; i < a.groups; ++i) {
                const double v = values[wv][i];
                ahead += (v > mine || (v == mine && i < g)) ? 1 : 0;
            }
            if (ahead >= a.top_groups) key[j] = 0;
        }
    }
    double sum = 0.0, mine = 0.0;
    int myid = 0;
    for (int i = 0; i < a.k; ++i) {
        uint64_t bk = 0;
        int bj = 0;
#pragma unroll
        for (int j = 0; j < NPL; ++j)
            if (key[j] > bk) { bk = key[j]; bj = j; }
        const uint64_t best = wave_max64(bk);
        const int e = int(wave_ext<false>(bk == best ? uint32_t(lane + 64 * bj) : 0xffffffffu));
        double s = 0.0;
#pragma unroll
        for (int j = 0; j < NPL; ++j)
            if (lane + 64 * j == e) {
                s = p[j];
                key[j] = 0;
            }
        s = __longlong_as_double(int64_t(readlane64(uint64_t(__double_as_longlong(s)), e & 63)));
        if (!a.sigmoid) s = s / denom;
        sum += s;
        if (lane == i) { mine = s; myid = e; }
    }
    if (here && lane < a.k) {
        const double w = a.renorm ? mine / (sum + 1e-20) : mine;
        a.ids[t * a.k + lane] = myid;
        a.w[t * a.k + lane] = float(w * double(a.scale));
    }
}

template <class T>
void score_type(const ScoreArgs& a, hipStream_t s, hipEvent_t stop) {
    const auto go = [&](auto kernel) {
        hipExtLaunchKernelGGL(kernel, dim3((a.T + 3) / 4), dim3(256), 0, s, nullptr, stop, 0, a);
    };
    if (a.n <= 64) go(score_route_kernel<T, 1>);
    else if (a.n <= 128) go(score_route_kernel<T, 2>);
    else if (a.n <= 256) go(score_route_kernel<T, 4>);
    else if (a.n <= 512) go(score_route_kernel<T, 8>);
    else go(score_route_kernel<T, 16>);
}

}  // namespace

hipError_t launch_score_route(const ScoreArgs& a, hipStream_t s, hipEvent_t stop) {
    if (a.T < 1 || a.n < 1 || a.n > kScoreMaxExperts || a.k < 1 || a.k > 16 || a.groups < 1 || a.n % a.groups ||
        a.top_groups < 1 || a.top_groups > a.groups || a.k > a.top_groups * (a.n / a.groups) || a.group_keys < 1 ||
        a.group_keys > 2 || (a.groups > 1 && a.group_keys > a.n / a.groups))
        return hipErrorInvalidValue;
    switch (a.type) {
    case kActF32: score_type<float>(a, s, stop); break;
    case kActF16: score_type<f16>(a, s, stop); break;
    case kActBF16: score_type<bf16>(a, s, stop); break;
    default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

}  // namespace xl::dev
