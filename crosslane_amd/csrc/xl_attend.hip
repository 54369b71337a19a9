// CDNA4 (gfx950) attention over a 4-bit cache. First form: a wave for each row and
// head, 64 tokens at a time, the running maximum and sum of one softmax.
#include <hip/hip_ext.h>

#include <algorithm>

#include "xl_act.hpp"
#include "xl_kv_index.hpp"

namespace xl {

AttendPlan attend_plan(int, int, int, int, int, int, int64_t) { return AttendPlan{}; }

namespace dev {
namespace {

template <class T, int D>
__global__ __launch_bounds__(64) void attend_kernel(AttendArgs a) {
    constexpr int C = D / 8, G = D / 32;
    __shared__ float q[D];
    __shared__ float prob[64];
    const KvBatch& b = a.b;
    const int h = blockIdx.x % a.q_heads, t = blockIdx.x / a.q_heads, lane = threadIdx.x;
    const int seq = seq_of(b, t);
    const SeqRows s = seq_rows(b, seq);
    if (s.bad) atomicOr(b.err, kDevErrBatch);
    if (t < s.first || t >= s.first + s.n) return;
    const int pos = s.len - s.n + (t - s.first), head = h / a.group;
    const Slab<D> slab(b.page);
    bool fine = true;
    for (int d = lane; d < D; d += 64) {
        q[d] = float(static_cast<const T*>(a.q)[int64_t(t) * a.q_stride + int64_t(h) * D + d]);
        fine = fine && fabsf(q[d]) <= 3.402823466e38f;
    }
    fine = __ballot(!fine) == 0;
    __syncthreads();
    float top = -INFINITY, sum = 0.0f, o[D / 64] = {};
    const int from = a.window ? max(0, pos - a.window + 1) : 0;
    for (int j0 = from & ~63; j0 <= pos; j0 += 64) {
        const int j = j0 + lane;
        int run = 0;
        const uint8_t* page = nullptr;
        if (j >= from && j <= pos) {
            const int64_t p = page_at(b, seq, uint32_t(j) >> 4, run);
            if (p >= 0) page = b.pages + p;
            else atomicOr(b.err, kDevErrBatch);
        }
        float x = -INFINITY;
        if (page) {
            const uint8_t* at = page + int64_t(head) * slab.bytes();
            const int tok = 16 * run + (j & 15);
            float dot = 0.0f;
            for (int c = 0; c < C; ++c) {
                const uint32_t w = reinterpret_cast<const uint32_t*>(at)[tok * C + (c & 3) * G + c / 4];
                const f16* e = reinterpret_cast<const f16*>(at + slab.k_scales()) + (tok * G + c / 4) * 2;
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    dot = fmaf(q[8 * c + k], fmaf(float(w >> (k / 2 * 4 + k % 2 * 16) & 15u), float(e[0]), float(e[1])), dot);
            }
            x = dot * a.scale;
            if (a.softcap > 0.0f) x = a.softcap * tanhf(x / a.softcap);
        }
        float m = x;
        for (int i = 32; i; i >>= 1) m = fmaxf(m, __shfl_xor(m, i));
        m = fmaxf(m, top);
        const float base = m == -INFINITY ? 0.0f : m;
        const float p = page ? expf(x - base) : 0.0f;
        float ps = p;
        for (int i = 32; i; i >>= 1) ps += __shfl_xor(ps, i);
        const float old = expf(top - base);
        sum = sum * old + ps;
        top = m;
        __syncthreads();
        prob[lane] = p;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < D / 64; ++i) o[i] *= old;
        for (int k = 0; k < 64; ++k) {
            const int jj = j0 + k;
            const uint64_t there = __ballot(page != nullptr);
            if (!(there >> k & 1)) continue;
            const uint64_t pg = __shfl(reinterpret_cast<unsigned long long>(page), k);
            const int tok = 16 * __shfl(run, k) + (jj & 15);
            const uint8_t* at = reinterpret_cast<const uint8_t*>(pg) + int64_t(head) * slab.bytes();
#pragma unroll
            for (int i = 0; i < D / 64; ++i) {
                const int d = lane + 64 * i;
                const uint16_t w = reinterpret_cast<const uint16_t*>(at + slab.v_codes())[(tok >> 2) * D + d / 8 * 8 + (tok >> 1 & 1) * 4 + (d / 4 & 1) * 2 + (tok & 1)];
                const f16* e = reinterpret_cast<const f16*>(at + slab.v_scales()) + ((tok >> 2) * G + d / 32) * 8 + (tok & 3);
                const float m2 = float(e[4]);
                o[i] = fmaf(prob[k], fmaf(float(w >> (4 * (d & 3)) & 15u), float(e[0]), m2), o[i]);
                if (e[0] != e[0]) sum = NAN;
            }
        }
    }
#pragma unroll
    for (int i = 0; i < D / 64; ++i) {
        const float y = !fine && pos >= 0 ? NAN : pos < 0 || sum == 0.0f ? 0.0f : o[i] / sum;
        static_cast<T*>(a.out)[int64_t(t) * a.out_stride + int64_t(h) * D + lane + 64 * i] = T(y);
    }
}

template <class T>
hipError_t attend_type(const AttendArgs& a, hipStream_t s, hipEvent_t stop) {
    const dim3 grid(uint32_t(a.b.rows) * uint32_t(a.q_heads));
    switch (a.b.dim) {
    case 64: hipExtLaunchKernelGGL((attend_kernel<T, 64>), grid, dim3(64), 0, s, nullptr, stop, 0, a); break;
    case 128: hipExtLaunchKernelGGL((attend_kernel<T, 128>), grid, dim3(64), 0, s, nullptr, stop, 0, a); break;
    case 256: hipExtLaunchKernelGGL((attend_kernel<T, 256>), grid, dim3(64), 0, s, nullptr, stop, 0, a); break;
    default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

}  // namespace

hipError_t launch_attend(const AttendArgs& a, hipStream_t s, hipEvent_t stop) {
    switch (a.type) {
    case kActF16: return attend_type<f16>(a, s, stop);
    case kActBF16: return attend_type<bf16>(a, s, stop);
    default: return hipErrorInvalidValue;
    }
}

}  // namespace dev
}  // namespace xl
