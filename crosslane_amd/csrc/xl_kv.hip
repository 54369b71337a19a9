// CDNA4 (gfx950) kernels that fill and read a cache of keys and values in 4 bits: rotary
// positions on q and k, groups of 32 values with a scale and a smallest value in
// float16, and the values back as floats.
//
// Bound by memory (4.2 TB/s of a write of 16384 rows, 4.7 of a read of 102000, as a copy). A
// thread has eight consecutive values of a head, so a group is four threads and a row 8, 16 or
// 32, joined by lane exchanges. Values are float32 between loads and codes; what is held is
// rounded as crosslane.h says, to the bit.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "xl_act.hpp"
#include "xl_kv_index.hpp"

namespace xl::dev {
namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ float quad_min(float v) {
    v = fminf(v, dpp_or<0xB1>(v, v));
    return fminf(v, dpp_or<0x4E>(v, v));
}
__device__ __forceinline__ float quad_max(float v) {
    v = fmaxf(v, dpp_or<0xB1>(v, v));
    return fmaxf(v, dpp_or<0x4E>(v, v));
}

// The first block looks at every sequence's starts and length.
__device__ __forceinline__ void check_batch(const KvBatch& b) {
    if (blockIdx.x == 0 && blockIdx.y == 0)
        for (int i = threadIdx.x; i < b.n_seqs; i += kThreads)
            if (seq_rows(b, i).bad) atomicOr(b.err, kDevErrBatch);
}

// Dims at ..+7 of a head's row x, turned. cs: cosine and sine of the token's angles.
template <class T, int D>
__device__ __forceinline__ void turned8(const T* x, int at, const KvRotary& r, const float2* cs, float (&v)[8]) {
    load8(x + at, 8, v);
    if (at >= 2 * r.n) return;
    if (r.interleaved) {
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            if (at + i >= 2 * r.n) break;
            const float2 f = cs[at / 2 + i / 2];
            const float a = v[i], b = v[i + 1];
            v[i] = a * f.x - b * f.y;
            v[i + 1] = b * f.x + a * f.y;
        }
    } else if (r.n % 8 == 0) {
        const bool second = at >= r.n;
        float w[8];
        load8(x + (second ? at - r.n : at + r.n), 8, w);
        const float2* f = cs + (second ? at - r.n : at);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = second ? v[i] * f[i].x + w[i] * f[i].y : v[i] * f[i].x - w[i] * f[i].y;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int d = at + i;
            if (d < r.n) v[i] = v[i] * cs[d].x - float(x[d + r.n]) * cs[d].y;
            else if (d < 2 * r.n) v[i] = v[i] * cs[d - r.n].x + float(x[d - r.n]) * cs[d - r.n].y;
        }
    }
}

// A block: one row, blockIdx.y of gridDim.y parts of its heads' chunks (q's heads, then k's, then v's), and the row's angles once.
// 91 us for 16384 rows of 32 + 16 heads of 128 (391 MB); stores past the caches and two or four blocks a row were no faster.
template <class T, int D>
__global__ __launch_bounds__(kThreads) void kv_write_kernel(KvBatch b, KvRotary r, KvRows x) {
    __shared__ float2 cs[D / 2];
    constexpr int C = D / 8;
    const int t = blockIdx.x;
    const int seq = seq_of(b, t);
    const SeqRows s = seq_rows(b, seq);
    check_batch(b);
    if (t < s.first || t >= s.first + s.n) return;
    const int pos = s.len - s.n + (t - s.first);
    if (r.n && pos >= 0) {
        for (int i = threadIdx.x; i < r.n; i += kThreads) {
            const int axis = i < r.end0 ? 0 : i < r.end1 ? 1 : 2;
            const int at = r.positions ? r.positions[axis * r.positions_stride + t] : pos;
            double sn, cn;
            sincos(double(at) * double(r.freqs[i]), &sn, &cn);
            cs[i] = make_float2(float(cn), float(sn));
        }
        __syncthreads();
    }
    const Slab<D> slab(b.page);
    int run = 0;
    const int64_t page = pos >= 0 ? page_at(b, seq, uint32_t(pos) >> 4, run) : -1;
    if (pos >= 0 && page < 0) atomicOr(b.err, kDevErrBatch);
    const int tok = 16 * run + (pos & 15);
    const int q_items = x.q ? x.q_heads * C : 0, items = q_items + 2 * b.kv_heads * C;
    for (int i = blockIdx.y * kThreads + threadIdx.x; i < items; i += gridDim.y * kThreads) {
        float v[8] = {};
        if (i < q_items) {
            if (pos >= 0) turned8<T, D>(static_cast<const T*>(x.q) + int64_t(t) * x.q_stride + i / C * D, i % C * 8, r, cs, v);
            store_rounded<T, 8>(static_cast<T*>(x.q_out) + int64_t(t) * x.q_out_stride + i * 8, 8, v);
            continue;
        }
        if (page < 0) continue;
        const int j = i - q_items, c = j % C;
        const bool is_v = j >= b.kv_heads * C;
        const int head = is_v ? j / C - b.kv_heads : j / C;
        if (is_v) load8(static_cast<const T*>(x.v) + int64_t(t) * x.v_stride + head * D + c * 8, 8, v);
        else turned8<T, D>(static_cast<const T*>(x.k) + int64_t(t) * x.k_stride + head * D, c * 8, r, cs, v);
        bool fine = true;
        float lo = 32768.0f, hi = -32768.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            fine = fine && fabsf(v[e]) <= 3.402823466e38f;
            v[e] = fminf(fmaxf(v[e], -32768.0f), 32768.0f);
            lo = fminf(lo, v[e]);
            hi = fmaxf(hi, v[e]);
        }
        // the lanes of this row (a wave has whole rows)
        const uint64_t row = ((1ull << C) - 1) << (threadIdx.x & 63 & ~(C - 1));
        fine = (__ballot(!fine) & row) == 0;
        const f16 m = f16(quad_min(lo));
        const f16 step = rounded<f16>(fmaxf((quad_max(hi) - float(m)) * (1.0f / 15.0f), 0.0f));   // (m may have been rounded up)
        const float inv = step > f16(0.0f) ? 1.0f / float(step) : 0.0f;
        uint32_t code[8];
#pragma unroll
        for (int e = 0; e < 8; ++e)
            code[e] = fine ? uint32_t(int(fminf(fmaxf(rintf((v[e] - float(m)) * inv), 0.0f), 15.0f))) : 0u;
        uint16_t mb = __builtin_bit_cast(uint16_t, m), sb = __builtin_bit_cast(uint16_t, step);
        if (!fine) {
            mb = sb = 0x7e00;
            if (c == 0) atomicOr(b.err, kDevErrNonFinite);
        }
        uint8_t* at = b.pages + page + int64_t(head) * slab.bytes();
        const int g = c / 4;
        if (!is_v) {
            uint32_t w = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) w |= code[2 * e] << (4 * e) | code[2 * e + 1] << (4 * e + 16);
            *reinterpret_cast<uint32_t*>(at + slab.k_word(tok, c)) = w;
            if ((c & 3) == 0) *reinterpret_cast<uint32_t*>(at + slab.k_scale(tok, g)) = uint32_t(sb) | uint32_t(mb) << 16;
        } else {
            uint16_t* o = reinterpret_cast<uint16_t*>(at + slab.v_half(tok, c));
            o[0] = uint16_t(code[0] | code[1] << 4 | code[2] << 8 | code[3] << 12);
            o[2] = uint16_t(code[4] | code[5] << 4 | code[6] << 8 | code[7] << 12);
            if ((c & 3) == 0) {
                uint16_t* e = reinterpret_cast<uint16_t*>(at + slab.v_scale(tok, g));
                e[0] = sb;
                e[4] = mb;
            }
        }
    }
}

// Many rows of a sequence (16 or more; 102000 rows 116 us, a row a block 190): a wave takes a run of 16 tokens of one head, with the widest loads that the cache's layout has (16 bytes
// of a token's key codes, of four tokens' value codes, and their scales). A sequence's runs that hold rows, from the run of its first row
// (below 0 where rows come before the first token), are numbered from starts[q] / 16 + 2q on: n rows lie in at most n / 16 + 2 runs.
template <class T, int D>
__global__ __launch_bounds__(kThreads) void kv_read_runs_kernel(KvBatch b, KvRows x) {
    constexpr int G = D / 32, C = D / 8, VP = D == 64 ? 1 : 2, VC = D == 256 ? 2 : 1;   // pairs of four tokens, and chunks, of a lane's values
    const int lane = threadIdx.x & 63;
    const uint32_t pair = 4 * blockIdx.x + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);   // a run's number and a head
    const int number = pair / uint32_t(b.kv_heads), head = pair - uint32_t(number) * uint32_t(b.kv_heads);
    check_batch(b);
    const auto first_number = [&](int q) { return (b.starts[q] >> 4) + 2 * q; };
    int seq = 0;
    for (int hi = b.n_seqs; hi - seq > 1;) {
        const int mid = (seq + hi) >> 1;
        if (first_number(mid) <= number) seq = mid;
        else hi = mid;
    }
    const SeqRows s = seq_rows(b, seq);
    const int first = s.len - s.n, run = (first >> 4) + number - first_number(seq);
    if (s.n == 0 || run < first >> 4 || run > (s.len - 1) >> 4) return;
    const Slab<D> slab(b.page);
    int in = 0;
    const int64_t page = run >= 0 ? page_at(b, seq, uint32_t(run), in) : -1;
    if (run >= 0 && page < 0 && lane == 0) atomicOr(b.err, kDevErrBatch);
    const uint8_t* at = b.pages + (page < 0 ? 0 : page) + int64_t(head) * slab.bytes();
    // the row of a token of the run (below 0 or from s.n on: none)
    const auto row_of = [&](int tok) { return 16 * run + tok - first; };
    const auto put = [&](void* out, int64_t stride, int tok, int d, const float (&v)[8]) {
        const int r = row_of(tok);
        if (r >= 0 && r < s.n) store8(static_cast<T*>(out) + int64_t(s.first + r) * stride + head * D + d, 8, v);
    };
    if (page < 0) {   // no tokens, or no page
        const float v[8] = {};
        for (int i = lane; i < 16 * C; i += 64) {
            put(x.k_out, x.k_stride, i / C, i % C * 8, v);
            put(x.v_out, x.v_stride, i / C, i % C * 8, v);
        }
        return;
    }
    const int k_tok = lane & 15, c = lane >> 4;
    uint32_t kc[G], ks[G], vc[VC][2 * VP], vs[4];
    const int v_quad = lane >> 4, v_chunk = D == 64 ? lane >> 1 & 7 : (lane & 15) * VC, v_pair = VP == 1 ? lane & 1 : 0;
    __builtin_memcpy(kc, __builtin_assume_aligned(at + 8 * D * in + 4 * (k_tok * C + c * G), G >= 4 ? 16 : 4 * G), sizeof kc);
    __builtin_memcpy(ks, __builtin_assume_aligned(at + slab.k_scale(16 * in + k_tok, 0), G >= 4 ? 16 : 4 * G), sizeof ks);
    __builtin_memcpy(vc, __builtin_assume_aligned(at + slab.v_codes() + 8 * D * in + 2 * (v_quad * D + v_chunk * 8) + 8 * v_pair, 8 * VP), sizeof vc);
    __builtin_memcpy(vs, __builtin_assume_aligned(at + slab.v_scale(16 * in + 4 * v_quad, v_chunk / 4), 16), sizeof vs);
    const auto half = [](uint32_t w, int i) { return float(__builtin_bit_cast(f16, uint16_t(i ? w >> 16 : w))); };
#pragma unroll
    for (int g = 0; g < G; ++g) {
        float v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = fmaf(float(kc[g] >> (k / 2 * 4 + k % 2 * 16) & 15u), half(ks[g], 0), half(ks[g], 1));
        put(x.k_out, x.k_stride, k_tok, 32 * g + 8 * c, v);
    }
#pragma unroll
    for (int u = 0; u < VC; ++u)
#pragma unroll
        for (int p = 0; p < VP; ++p)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int pair = VP == 1 ? v_pair : p;
                const uint32_t step = VP == 1 ? (v_pair ? vs[1] : vs[0]) : vs[p], small = VP == 1 ? (v_pair ? vs[3] : vs[2]) : vs[2 + p];
                float v[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) v[k] = fmaf(float(vc[u][2 * p + k / 4] >> (16 * e + k % 4 * 4) & 15u), half(step, e), half(small, e));
                put(x.v_out, x.v_stride, 4 * v_quad + 2 * pair + e, 8 * (v_chunk + u), v);
            }
}

// Few rows of each: a block has one row, blockIdx.y of gridDim.y parts of its heads' chunks (keys, then values).
template <class T, int D>
__global__ __launch_bounds__(kThreads) void kv_read_kernel(KvBatch b, KvRows x) {
    constexpr int C = D / 8;
    const int t = blockIdx.x;
    const int seq = seq_of(b, t);
    const SeqRows s = seq_rows(b, seq);
    check_batch(b);
    if (t < s.first || t >= s.first + s.n) return;
    const int pos = s.len - s.n + (t - s.first);
    const Slab<D> slab(b.page);
    int run = 0;
    const int64_t page = pos >= 0 ? page_at(b, seq, uint32_t(pos) >> 4, run) : -1;
    if (pos >= 0 && page < 0) atomicOr(b.err, kDevErrBatch);
    const int tok = 16 * run + (pos & 15);
    for (int i = blockIdx.y * kThreads + threadIdx.x; i < 2 * b.kv_heads * C; i += gridDim.y * kThreads) {
        const bool is_v = i >= b.kv_heads * C;
        const int j = is_v ? i - b.kv_heads * C : i, head = j / C, c = j % C, g = c / 4;
        float v[8] = {};
        if (page >= 0) {
            const uint8_t* at = b.pages + page + int64_t(head) * slab.bytes();
            if (!is_v) {
                const uint32_t w = *reinterpret_cast<const uint32_t*>(at + slab.k_word(tok, c));
                const f16* e = reinterpret_cast<const f16*>(at + slab.k_scale(tok, g));
                const float step = float(e[0]), m = float(e[1]);
#pragma unroll
                for (int k = 0; k < 8; ++k) v[k] = fmaf(float(w >> (k / 2 * 4 + k % 2 * 16) & 15u), step, m);
            } else {
                const uint16_t* o = reinterpret_cast<const uint16_t*>(at + slab.v_half(tok, c));
                const f16* e = reinterpret_cast<const f16*>(at + slab.v_scale(tok, g));
                const uint32_t w = o[0] | uint32_t(o[2]) << 16;
                const float step = float(e[0]), m = float(e[4]);
#pragma unroll
                for (int k = 0; k < 8; ++k) v[k] = fmaf(float(w >> (4 * k) & 15u), step, m);
            }
        }
        store8(is_v ? static_cast<T*>(x.v_out) + int64_t(t) * x.v_stride + j * 8 : static_cast<T*>(x.k_out) + int64_t(t) * x.k_stride + j * 8,
               8, v);
    }
}

// Few rows: a thread for each chunk, so that one token is one step; many: a block for each row.
int parts(int rows, int items) { return rows >= 512 ? 1 : std::min((items + kThreads - 1) / kThreads, std::max(1, 1024 / rows)); }

template <class T, int D>
hipError_t write_go(const KvBatch& b, const KvRotary& r, const KvRows& x, hipStream_t s) {
    const int items = ((x.q ? x.q_heads : 0) + 2 * b.kv_heads) * (D / 8);
    hipLaunchKernelGGL((kv_write_kernel<T, D>), dim3(b.rows, parts(b.rows, items)), dim3(kThreads), 0, s, b, r, x);
    return hipGetLastError();
}
template <class T, int D>
hipError_t read_go(const KvBatch& b, const KvRows& x, hipStream_t s) {
    if (b.max_rows >= 16) {
        const int64_t pairs = ((int64_t(b.rows) >> 4) + 2 * int64_t(b.n_seqs)) * b.kv_heads;
        if (pairs < int64_t(1) << 26) {   // (a launch counts threads in 32 bits)
            hipLaunchKernelGGL((kv_read_runs_kernel<T, D>), dim3(uint32_t((pairs + 3) / 4)), dim3(kThreads), 0, s, b, x);
            return hipGetLastError();
        }
    }
    const int items = 2 * b.kv_heads * (D / 8);
    hipLaunchKernelGGL((kv_read_kernel<T, D>), dim3(b.rows, parts(b.rows, items)), dim3(kThreads), 0, s, b, x);
    return hipGetLastError();
}
template <class F>
hipError_t by_type_and_dim(int type, int dim, F&& f) {
    const auto dims = [&](auto t) {
        using T = decltype(t);
        switch (dim) {
        case 64: return f.template operator()<T, 64>();
        case 128: return f.template operator()<T, 128>();
        case 256: return f.template operator()<T, 256>();
        default: return hipErrorInvalidValue;
        }
    };
    switch (type) {
    case kActF32: return dims(float());
    case kActF16: return dims(f16());
    case kActBF16: return dims(bf16());
    default: return hipErrorInvalidValue;
    }
}

}  // namespace

hipError_t launch_kv_write(const KvBatch& b, const KvRotary& r, const KvRows& x, hipStream_t s) {
    if (r.n > b.dim / 2) return hipErrorInvalidValue;
    return by_type_and_dim(x.type, b.dim, [&]<class T, int D>() { return write_go<T, D>(b, r, x, s); });
}
hipError_t launch_kv_read(const KvBatch& b, const KvRows& x, hipStream_t s) {
    return by_type_and_dim(x.type, b.dim, [&]<class T, int D>() { return read_go<T, D>(b, x, s); });
}

}  // namespace xl::dev
