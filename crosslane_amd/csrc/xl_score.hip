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
constexpr float kMaxFloat = 3.402823466e38f;

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
__device__ __forceinline__ double readlane_f64(double v, int lane) {
    return __longlong_as_double(int64_t(readlane64(uint64_t(__double_as_longlong(v)), lane)));
}
__device__ __forceinline__ double wave_sum64(double x) {
    const auto add = [](double v, uint64_t o) { return v + __longlong_as_double(int64_t(o)); };
    const auto bits = [](double v) { return uint64_t(__double_as_longlong(v)); };
    x = add(x, dpp64<0xB1>(bits(x)));
    x = add(x, dpp64<0x4E>(bits(x)));
    x = add(x, dpp64<0x141>(bits(x)));
    x = add(x, dpp64<0x140>(bits(x)));
    x = add(x, dpp64<0x142, 0xA>(bits(x)));
    x = add(x, dpp64<0x143, 0xC>(bits(x)));
    return readlane_f64(x, 63);
}
// The largest / smallest of the wave. Lanes that a step leaves out get the identity:
// so each step is one instruction.
template <bool MAX>
__device__ __forceinline__ uint32_t wave_top(uint32_t v) {
    constexpr int id = MAX ? 0 : -1;
    const auto f = [](uint32_t x, uint32_t y) { return MAX ? max(x, y) : min(x, y); };
    v = f(v, uint32_t(__builtin_amdgcn_update_dpp(id, int(v), 0xB1, 0xF, 0xF, false)));   // quad_perm 1,0,3,2
    v = f(v, uint32_t(__builtin_amdgcn_update_dpp(id, int(v), 0x4E, 0xF, 0xF, false)));   // quad_perm 2,3,0,1
    v = f(v, uint32_t(__builtin_amdgcn_update_dpp(id, int(v), 0x141, 0xF, 0xF, false)));  // row_half_mirror
    v = f(v, uint32_t(__builtin_amdgcn_update_dpp(id, int(v), 0x140, 0xF, 0xF, false)));  // row_mirror
    v = f(v, uint32_t(__builtin_amdgcn_update_dpp(id, int(v), 0x142, 0xA, 0xF, false)));  // row_bcast:15
    v = f(v, uint32_t(__builtin_amdgcn_update_dpp(id, int(v), 0x143, 0xC, 0xF, false)));  // row_bcast:31
    return uint32_t(__builtin_amdgcn_readlane(int(v), 63));
}
// An expert's score, 0 where it is masked (softmax: times the sum of these; `largest`
// is finite). Without branches, so that the slots' exps run in step.
__device__ __forceinline__ double sigmoid(float l) { return 1.0 / (1.0 + exp(-double(l))); }
__device__ __forceinline__ double part(float l, double largest) { return exp(double(l) - largest); }
// a where m is all ones, b where it is zero.
__device__ __forceinline__ uint32_t pick(uint32_t m, uint32_t a, uint32_t b) { return (a & m) | (b & ~m); }
__device__ __forceinline__ uint64_t pick(uint32_t m, uint64_t a, uint64_t b) {
    return uint64_t(pick(m, uint32_t(a), uint32_t(b))) | uint64_t(pick(m, uint32_t(a >> 32), uint32_t(b >> 32))) << 32;
}
__device__ __forceinline__ uint64_t max64(uint64_t a, uint64_t b) { return a > b ? a : b; }
__device__ __forceinline__ uint64_t min64(uint64_t a, uint64_t b) { return a > b ? b : a; }

// The two largest keys of each aligned run of `lanes` (1, 2, ... 64) lanes, in all of
// them, from each lane's two.
__device__ __forceinline__ void top_two(uint64_t& m1, uint64_t& m2, int lanes) {
    const auto join = [&](uint64_t o1, uint64_t o2) {
        m2 = max64(min64(m1, o1), max64(m2, o2));
        m1 = max64(m1, o1);
    };
    if (lanes >= 2) join(dpp64<0xB1>(m1), dpp64<0xB1>(m2));
    if (lanes >= 4) join(dpp64<0x4E>(m1), dpp64<0x4E>(m2));
    if (lanes >= 8) join(dpp64<0x141>(m1), dpp64<0x141>(m2));
    if (lanes >= 16) join(dpp64<0x140>(m1), dpp64<0x140>(m2));
    if (lanes >= 32) join(__shfl_xor(static_cast<unsigned long long>(m1), 16), __shfl_xor(static_cast<unsigned long long>(m2), 16));
}

// One wave per token. Up to 64 groups: each has a run of 64 / (groups rounded up to a
// power of two) lanes, its experts going round them (one group: all 64), so that its
// value is a few lane steps away and ranks come from lanes' values as scalars. MANY
// (more groups): experts go round all lanes, and groups' keys and values through LDS.
//
// Bound by instructions: 800 for 256 experts in 8 groups and 8 picks, a third of them the
// scores' (exp and a quotient in double), which at 8192 tokens is 10.6 of the 14.0 us. A
// pick is a maximum of the keys' upper words over the wave; only where two lanes have the
// same do lower words and indexes decide.
template <class T, int NPL, bool MANY>
__global__ __launch_bounds__(256) void score_route_kernel(ScoreArgs a) {
    constexpr int WAVES = 4;
    __shared__ uint64_t keys[MANY ? WAVES : 1][MANY ? NPL * 64 : 1];
    __shared__ double values[MANY ? WAVES : 1][MANY ? NPL * 64 : 1];
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t t = int64_t(blockIdx.x) * WAVES + wv;
    const bool here = t < a.T;
    if (!MANY && !here) return;   // MANY: every wave reaches the barriers
    const T* lg = static_cast<const T*>(a.logits) + (here ? t : 0) * a.stride;
    const int size = a.size, run = MANY ? 64 : 1 << a.run;   // a group's experts and lanes
    const int g = MANY ? 0 : lane >> a.run, r = lane & (run - 1);
    const int first = MANY ? r : g < a.groups ? g * size + r : a.n;   // the lane's experts: first, first + run, ...
    const int end = MANY ? a.n : g < a.groups ? (g + 1) * size : 0;   // ... below end
    float l[NPL];
    float b[NPL];
    float top = -__int_as_float(0x7f800000);
    bool bad = false;
#pragma unroll
    for (int j = 0; j < NPL; ++j) {
        const int e = first + run * j, at = min(e, a.n - 1);
        l[j] = float(lg[at]);
        b[j] = a.bias ? a.bias[at] : 0.0f;
    }
#pragma unroll
    for (int j = 0; j < NPL; ++j) {
        const bool in = first + run * j < end, no = !(l[j] <= kMaxFloat) || !(fabsf(b[j]) <= kMaxFloat);
        bad |= in && no;
        l[j] = !in ? -__int_as_float(0x7f800000) : no ? 0.0f : l[j];   // picks stay indexes of experts
        b[j] = no ? 0.0f : b[j];
        top = fmaxf(top, l[j]);
    }
    if (__any(bad) && here && lane == 0) atomicOr(a.err, kDevErrNonFinite);
    double p[NPL], denom = 1.0, largest = 0.0;
    if (a.sigmoid) {
#pragma unroll
        for (int j = 0; j < NPL; ++j) p[j] = sigmoid(l[j]);
    } else {
        // the largest logit, by integers that order as floats do
        const uint32_t ot = wave_top<true>(ordered(top));
        largest = double(fmaxf(__uint_as_float((ot & 0x80000000u) ? (ot ^ 0x80000000u) : ~ot), -kMaxFloat));
        double total = 0.0;
#pragma unroll
        for (int j = 0; j < NPL; ++j) {
            p[j] = part(l[j], largest);
            total += p[j];
        }
        denom = wave_sum64(total);
        denom = denom > 0.0 ? denom : 1.0;
#pragma unroll
        for (int j = 0; j < NPL; ++j) p[j] = p[j] / denom;
    }
    uint64_t key[NPL];
#pragma unroll
    for (int j = 0; j < NPL; ++j)
        key[j] = first + run * j < end ? ordered64(l[j] >= -kMaxFloat ? p[j] + double(b[j]) : kMaskedKey) : 0;
    if constexpr (MANY) {
#pragma unroll
        for (int j = 0; j < NPL; ++j) keys[wv][lane + 64 * j] = key[j];
        __syncthreads();
        for (int i = lane; i < a.groups; i += 64) {
            uint64_t m1 = 0, m2 = 0;
            for (int e = i * size; e < (i + 1) * size; ++e) {
                const uint64_t v = keys[wv][e];
                m2 = max64(m2, min64(m1, v));
                m1 = max64(m1, v);
            }
            values[wv][i] = unordered64(m1) + (a.group_keys == 2 ? unordered64(m2) : 0.0);
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < NPL; ++j) {
            if (lane + 64 * j >= a.n) continue;
            const int mine = (lane + 64 * j) / size;
            int ahead = 0;
            for (int i = 0; i < a.groups; ++i)
                ahead += values[wv][i] > values[wv][mine] || (values[wv][i] == values[wv][mine] && i < mine) ? 1 : 0;
            if (ahead >= a.top_groups) key[j] = 0;
        }
    } else if (a.top_groups < a.groups) {
        uint64_t m1 = 0, m2 = 0;
#pragma unroll
        for (int j = 0; j < NPL; ++j) {
            m2 = max64(m2, min64(m1, key[j]));
            m1 = max64(m1, key[j]);
        }
        top_two(m1, m2, run);
        const double value = unordered64(m1) + (a.group_keys == 2 ? unordered64(m2) : 0.0);
        int ahead = 0;   // a group stays if fewer than top_groups are ahead of it
        for (int i = 0; i < a.groups; ++i) {
            const double v = readlane_f64(value, i * run);
            ahead += v > value || (v == value && i < g) ? 1 : 0;
        }
        if (ahead >= a.top_groups)
#pragma unroll
            for (int j = 0; j < NPL; ++j) key[j] = 0;
    }
    // Up to 8 slots: each lane's keys in order first (neighbours change places, so that
    // equal ones keep theirs), and a pick is the best of the lanes' first ones.
    constexpr bool SORTED = NPL <= 8;
    uint32_t slot[NPL];
#pragma unroll
    for (int j = 0; j < NPL; ++j) slot[j] = j;
    if constexpr (SORTED)
#pragma unroll
        for (int n = NPL - 1; n > 0; --n)
#pragma unroll
            for (int j = 0; j < n; ++j) {
                const uint32_t swap = key[j] < key[j + 1] ? ~0u : 0u;
                const uint64_t k0 = key[j], k1 = key[j + 1];
                const uint32_t s0 = slot[j], s1 = slot[j + 1];
                key[j] = pick(swap, k1, k0);
                key[j + 1] = pick(swap, k0, k1);
                slot[j] = pick(swap, s1, s0);
                slot[j + 1] = pick(swap, s0, s1);
            }
    int myid = 0;
    for (int i = 0; i < a.k; ++i) {
        uint64_t bk = key[0];
        uint32_t be = slot[0];
        if constexpr (!SORTED)
#pragma unroll
            for (int j = 1; j < NPL; ++j) {
                const bool more = key[j] > bk;
                bk = more ? key[j] : bk;
                be = more ? uint32_t(j) : be;
            }
        const uint32_t hi = uint32_t(bk >> 32), best = wave_top<true>(hi);
        uint64_t who = __ballot(hi == best);
        if (who & (who - 1)) {
            const uint32_t lo = wave_top<true>(hi == best ? uint32_t(bk) : 0u);
            const bool in = hi == best && uint32_t(bk) == lo;
            const uint32_t e = uint32_t(first) + uint32_t(run) * be;
            const uint32_t least = wave_top<false>(in ? e : 0xffffffffu);   // all lanes take part
            who = __ballot(in && e == least);
        }
        const int from = __builtin_ctzll(who);
        const uint32_t taken = lane == from ? ~0u : 0u;
        if constexpr (SORTED) {
#pragma unroll
            for (int j = 0; j + 1 < NPL; ++j) {
                key[j] = pick(taken, key[j + 1], key[j]);
                slot[j] = pick(taken, slot[j + 1], slot[j]);
            }
            key[NPL - 1] = pick(taken, uint64_t(0), key[NPL - 1]);
        } else {
#pragma unroll
            for (int j = 0; j < NPL; ++j) key[j] = taken && uint32_t(j) == be ? 0 : key[j];
        }
        const int e = __builtin_amdgcn_readlane(first + run * int(be), from);
        if (lane == i) myid = e;
    }
    // the picks' scores again, all at once
    double s = 0.0;
    if (lane < a.k) {
        const float x = float(lg[myid]), at = x <= kMaxFloat ? x : 0.0f;
        s = a.sigmoid ? sigmoid(at) : part(at, largest) / denom;
    }
    const double sum = wave_sum64(s);
    if (here && lane < a.k) {
        const double w = a.renorm ? s / (sum + 1e-20) : s;
        a.ids[t * a.k + lane] = myid;
        a.w[t * a.k + lane] = float(w * double(a.scale));
    }
}

template <class T>
void score_type(ScoreArgs a, hipStream_t s, hipEvent_t stop) {
    const auto go = [&](auto kernel) {
        hipExtLaunchKernelGGL(kernel, dim3((a.T + 3) / 4), dim3(256), 0, s, nullptr, stop, 0, a);
    };
    a.size = a.n / a.groups;
    if (a.groups > 64) return go(score_route_kernel<T, 16, true>);
    for (a.run = 6; a.groups << a.run > 64;) --a.run;
    const int slots = (a.size + (1 << a.run) - 1) >> a.run;
    if (slots <= 1) go(score_route_kernel<T, 1, false>);
    else if (slots <= 2) go(score_route_kernel<T, 2, false>);
    else if (slots <= 4) go(score_route_kernel<T, 4, false>);
    else if (slots <= 6) go(score_route_kernel<T, 6, false>);
    else if (slots <= 8) go(score_route_kernel<T, 8, false>);
    else if (slots <= 16) go(score_route_kernel<T, 16, false>);
    else go(score_route_kernel<T, 32, false>);   // a number of groups far from a power of two
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
