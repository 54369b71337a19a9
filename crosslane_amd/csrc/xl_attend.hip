// CDNA4 (gfx950) attention over a 4-bit cache.
//
//   out = sum_j p_j v_j / sum_j p_j,   p_j = exp(x_j - m),   x_j = scale * q . k_j
//
// One pass over the tokens: m is a maximum so far, and where a later one passes it by more
// than 2^8 in weight, what was summed is scaled down. Codes of 4 bits become float16 by two
// instructions a pair (bits under an exponent, and that exponent's value off again) and their
// scale and smallest value by one fused multiply-add, rounded to float16 once: half a step
// of 2^-11, an eighth of what bfloat16 outputs round away and as much as float16 ones do.
#include <hip/hip_ext.h>

#include <algorithm>

#include "xl_act.hpp"
#include "xl_format.hpp"
#include "xl_kv_index.hpp"

namespace xl {
namespace {

constexpr int kSplitTokens = 256; // the least tokens that are worth a workgroup of their own

}  // namespace

// Splits: as many workgroups as fill the card four times (1024), where each has kSplitTokens at least.
AttendPlan attend_plan(int dim, int kv_heads, int q_heads, int n_seqs, int rows, int max_rows, int64_t max_tokens) {
    AttendPlan p;
    const int group = q_heads / kv_heads;
    const int64_t most = int64_t(max_rows) * group;
    p.tiles = int((most + 15) / 16);
    const int64_t wgs = int64_t(n_seqs) * kv_heads * p.tiles;
    const int64_t want = (1024 + wgs - 1) / wgs, can = (max_tokens + kSplitTokens - 1) / kSplitTokens;
    p.splits = int(std::max<int64_t>(1, std::min<int64_t>(128, std::min(want, can))));
    p.groups = std::max(wgs * p.splits, int64_t(rows) * q_heads);
    if (p.splits > 1) {
        const uint64_t parts = uint64_t(rows) * uint64_t(q_heads) * uint64_t(p.splits);
        p.part_ml = align256(parts * uint64_t(dim) * 4);
        p.bytes = p.part_ml + align256(parts * 8);
    }
    return p;
}

namespace dev {
namespace {

typedef f16 h2 __attribute__((ext_vector_type(2)));
typedef f16 h8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

constexpr float kLowest = -3.402823466e38f;   // a maximum before any token (below every score but -inf)
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLazy = 8.0f;                 // weights up to 2^8 before the maximum moves (float16 holds 2^15)

__device__ __forceinline__ h2 as_h2(uint32_t v) { return __builtin_bit_cast(h2, v); }
__device__ __forceinline__ uint32_t as_u32(h2 v) { return __builtin_bit_cast(uint32_t, v); }
__device__ __forceinline__ h2 both(f16 v) { return h2{v, v}; }

// Nibbles 0 and 4, 1 and 5, 2 and 6, 3 and 7 of a word, as pairs of whole numbers in float16: a nibble
// under the exponent of 1024 is 1024 + code, four bits higher under that of 64 it is 64 + code.
__device__ __forceinline__ void codes8(uint32_t w, h2 (&c)[4]) {
    const uint32_t u = w >> 8;
    c[0] = as_h2((w & 0x000f000fu) | 0x64006400u) - both(f16(1024.0f));
    c[1] = as_h2((w & 0x00f000f0u) | 0x54005400u) - both(f16(64.0f));
    c[2] = as_h2((u & 0x000f000fu) | 0x64006400u) - both(f16(1024.0f));
    c[3] = as_h2((u & 0x00f000f0u) | 0x54005400u) - both(f16(64.0f));
}
__device__ __forceinline__ h8 join(h2 a, h2 b, h2 c, h2 d) {
    return __builtin_bit_cast(h8, u4{as_u32(a), as_u32(b), as_u32(c), as_u32(d)});
}
__device__ __forceinline__ f4 mfma16(h8 a, h8 b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

// The largest of four pairs of float16 as bit patterns without sign: 0x7c00 and above are no numbers.
__device__ __forceinline__ uint32_t worst(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    constexpr uint32_t M = 0x7fff7fffu;
    typedef uint16_t s2 __attribute__((ext_vector_type(2)));
    const auto most = [](s2 x, s2 y) { return __builtin_elementwise_max(x, y); };
    const auto v = [](uint32_t x) { return __builtin_bit_cast(s2, x & M); };
    const s2 m = most(most(v(a), v(b)), most(v(c), v(d)));
    return max(uint32_t(m[0]), uint32_t(m[1]));
}
// Maximum / sum over the four runs of 16 lanes, in every lane.
__device__ __forceinline__ float rows_max(float v) {
    v = fmaxf(v, __shfl_xor(v, 16));
    return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float rows_sum(float v) {
    v += __shfl_xor(v, 16);
    return v + __shfl_xor(v, 32);
}
// softcap * tanh(x / softcap), times log2(e): tanh y = 1 - 2 / (exp(2 y) + 1), within 2^-22 of 1.
struct Cap {
    float in, out;   // 2 log2(e) / softcap, softcap * log2(e)
    __device__ __forceinline__ float operator()(float x) const {
        return out * (1.0f - 2.0f * __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(x * in) + 1.0f));
    }
};

// Rows of q in float16. A bfloat16 row is taken times a power of two that brings its largest value to 1..2, so
// that float16 holds all its bits, down to 2^-25 of that value; `up` is that power's inverse. A row with a value that is not
// finite is 0 here and `bad`.
template <class T>
__device__ __forceinline__ int row_exponent(float top) {
    if (sizeof(T) == 2 && __is_same(T, f16)) return 0;
    return top > 0.0f && top <= 3.402823466e38f ? __builtin_amdgcn_frexp_expf(top) - 1 : 0;
}

// What a lane loads of a tile of 32 tokens (two runs of 16), for keys as the first operand of the scores
// (token lane % 16 of each run, the eight dims 32g + 8c with c = lane / 16 of every group g), and for values as
// the first operand of the outputs (dims D / 16 * (lane % 16) on, the four tokens 4c of each run).
template <int D>
struct TileLoads {
    static constexpr int G = D / 32;
    uint32_t kc[2][G], ks[2][G], vc[2][D >= 128 ? D / 32 : 4];
    u4 vs[2];
    template <int N>
    static __device__ __forceinline__ void load(const uint8_t* p, uint32_t (&w)[N]) {
        __builtin_memcpy(w, __builtin_assume_aligned(p, N >= 4 ? 16 : 4 * N), 4 * N);
    }
    __device__ __forceinline__ void keys(int i, const uint8_t* slab, const Slab<D>& s, int run, int lane) {
        const int tok = 16 * run + (lane & 15);
        load(slab + 4 * (tok * (D / 8) + (lane >> 4) * G), kc[i]);
        load(slab + s.k_scale(tok, 0), ks[i]);
    }
    __device__ __forceinline__ void values(int i, const uint8_t* slab, const Slab<D>& s, int run, int lane) {
        const int quad = 4 * run + (lane >> 4), chunk = D >= 128 ? (lane & 15) * (D / 128) : (lane & 15) >> 1;
        load(slab + s.v_codes() + 2 * (quad * D + chunk * 8), vc[i]);
        __builtin_memcpy(&vs[i], __builtin_assume_aligned(slab + s.v_scales() + 16 * (quad * G + chunk / 4), 16), 16);
    }
};

// Few rows (of one sequence and kv head: its tokens' rows, each with `group` heads): a workgroup has 16 of them and
// one of `splits` parts of the tokens, its four waves every fourth tile of 32.
//
// Bound by the cache's bytes. A wave makes score^T = K q^T and out^T = V^T p^T with
// v_mfma_f32_16x16x32_f16: keys and values go from memory to registers and from there into the matrix cores as the
// first operand, with no LDS and no exchange between lanes; the scores come out in the lanes (row lane % 16, tokens
// 4 (lane / 16) ..+3 of each run) where the second product wants its weights, since the order of tokens
// within its sum is free. Loads of the next tile follow the last use of this one's registers.
template <class T, int D>
__global__ __launch_bounds__(256, D == 256 ? 2 : 4) void attend_few_kernel(AttendArgs a) {
    constexpr int G = D / 32, N = D / 16;
    __shared__ float part[4][16][D + 4];
    __shared__ float top_sh[4][16], sum_sh[4][16];
    const KvBatch& b = a.b;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane >> 4;
    uint32_t at = blockIdx.x;
    const int head = at % b.kv_heads;
    at /= b.kv_heads;
    const int split = at % a.splits;
    at /= a.splits;
    const int tile = at % a.tiles, seq = at / a.tiles;
    const SeqRows s = seq_rows(b, seq);
    if (s.bad && threadIdx.x == 0) atomicOr(b.err, kDevErrBatch);
    const int row0 = 16 * tile, rows = min(16, s.n * a.group - row0);
    if (rows <= 0) return;
    // this lane's row, and the tokens that it sees: lo ..hi - 1
    const int row = row0 + min(lane & 15, rows - 1), row_t = row / a.group, row_h = head * a.group + row - row_t * a.group;
    const int before = s.len - s.n;
    const int hi = before + row_t + 1, lo = a.window ? max(0, hi - a.window) : 0;
    // ... the least and the most of the 16 rows
    const int first_t = row0 / a.group, last_t = (row0 + rows - 1) / a.group;
    const int lo_all = a.window ? max(0, before + first_t + 1 - a.window) : 0, hi_all = before + last_t + 1;
    const int lo_most = a.window ? max(0, before + last_t + 1 - a.window) : 0, hi_least = before + first_t + 1;
    const int tile0 = lo_all >> 5, tiles = hi_all > lo_all ? ((hi_all + 31) >> 5) - tile0 : 0;
    const int per = max(kSplitTokens / 32, ((tiles + a.splits - 1) / a.splits + 3) & ~3);
    const int begin = tile0 + split * per + wave, end = tile0 + min(tiles, (split + 1) * per);

    const Slab<D> slab(b.page);
    const uint8_t* base = b.pages + int64_t(head) * slab.bytes();
    const int last_run = (hi_all - 1) >> 4;
    TileLoads<D> t;
    // a run's page (of the last one where the tile's second run lies behind it); a bad page's tokens are hidden
    const auto page = [&](int run, int& in, bool& ok) {
        const int64_t p = page_at(b, seq, uint32_t(min(run, last_run)), in);
        ok = p >= 0;
        return base + (ok ? p : 0);
    };
    const uint8_t* pg[2];
    int in[2];
    bool ok[2];
    if (begin < end) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            pg[i] = page(2 * begin + i, in[i], ok[i]);
            t.keys(i, pg[i], slab, in[i], lane);
            t.values(i, pg[i], slab, in[i], lane);
        }
    }

    // q: the second operand, row lane % 16, dims 32g + 8c ..+7
    h8 q[G];
    bool bad;
    float up;
    {
        const T* p = static_cast<const T*>(a.q) + int64_t(s.first + row_t) * a.q_stride + int64_t(row_h) * D + 8 * c;
        float v[G][8], m = 0.0f;
#pragma unroll
        for (int g = 0; g < G; ++g) {
            load8(p + 32 * g, 8, v[g]);
            m = amax8(v[g], m);
        }
        m = rows_max(m);
        bad = m > 3.402823466e38f;
        const int e = row_exponent<T>(m);
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
            for (int i = 0; i < 8; ++i) q[g][i] = bad ? f16(0.0f) : f16(__builtin_amdgcn_ldexpf(v[g][i], -e));
        up = __builtin_amdgcn_ldexpf(a.softcap > 0.0f ? a.scale : a.scale * kLog2e, e);
    }
    const Cap cap{2.0f * kLog2e / a.softcap, a.softcap * kLog2e};

    float top = kLowest, sum = 0.0f;
    f4 o[N] = {};
    for (int tl = begin; tl < end; tl += 4) {
        const bool more = tl + 4 < end;
        const bool ok0 = ok[0], ok1 = ok[1];
        if (more) {
#pragma unroll
            for (int i = 0; i < 2; ++i) pg[i] = page(2 * (tl + 4) + i, in[i], ok[i]);
        }
        float x[8];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            f4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int g = 0; g < G; ++g) {
                const h2 sm = as_h2(t.ks[i][g]), step = both(sm[0]), small = both(sm[1]);
                h2 k[4];
                codes8(t.kc[i][g], k);
#pragma unroll
                for (int j = 0; j < 4; ++j) k[j] = __builtin_elementwise_fma(k[j], step, small);
                acc = mfma16(join(k[0], k[1], k[2], k[3]), q[g], acc);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) x[4 * i + j] = acc[j] * up;
        }
        if (more) {
#pragma unroll
            for (int i = 0; i < 2; ++i) t.keys(i, pg[i], slab, in[i], lane);
        }
        if (a.softcap > 0.0f) {
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = cap(x[j]);
        }
        // the first and last tiles hide tokens from some rows; what no row sees may be anything
        if (32 * tl < lo_most || 32 * tl + 32 > hi_least || !(ok0 && ok1)) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int tok = 32 * tl + 16 * (j >> 2) + 4 * c + (j & 3);
                const bool there = j < 4 ? ok0 : ok1;
                if (tok < lo || tok >= hi || !there) x[j] = -INFINITY;
                if (tok >= hi_all || !there) {
                    uint32_t& w0 = reinterpret_cast<uint32_t*>(&t.vs[j >> 2])[(j & 3) >> 1];
                    uint32_t& w1 = reinterpret_cast<uint32_t*>(&t.vs[j >> 2])[2 + ((j & 3) >> 1)];
                    w0 &= j & 1 ? 0x0000ffffu : 0xffff0000u;
                    w1 &= j & 1 ? 0x0000ffffu : 0xffff0000u;
                }
            }
            if (lane == 0 && !(ok0 && ok1)) atomicOr(b.err, kDevErrBatch);
        }
        float m = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
        if (__any(m > top + kLazy)) {
            m = fmaxf(rows_max(m), top);
            const float f = __builtin_amdgcn_exp2f(top - m);
            top = m;
            sum *= f;
#pragma unroll
            for (int n = 0; n < N; ++n) o[n] *= f;
        }
        float p[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            p[j] = __builtin_amdgcn_exp2f(x[j] - top);
            sum += p[j];
        }
        // a token held as NaN: its values as 0, and the rows that see it NaN by their sum
        {
            const uint32_t w = worst(t.vs[0][0], t.vs[0][1], t.vs[1][0], t.vs[1][1]);
            if (__any(w >= 0x7c00u)) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    uint32_t& w0 = reinterpret_cast<uint32_t*>(&t.vs[j >> 2])[(j & 3) >> 1];
                    uint32_t& w1 = reinterpret_cast<uint32_t*>(&t.vs[j >> 2])[2 + ((j & 3) >> 1)];
                    const uint32_t e = (j & 1 ? w0 >> 16 : w0) & 0x7fffu;
                    if (e >= 0x7c00u) {
                        w0 &= j & 1 ? 0x0000ffffu : 0xffff0000u;
                        w1 &= j & 1 ? 0x0000ffffu : 0xffff0000u;
                        if (x[j] != -INFINITY) sum = NAN;
                    }
                }
            }
        }
        const h8 w = {f16(p[0]), f16(p[1]), f16(p[2]), f16(p[3]), f16(p[4]), f16(p[5]), f16(p[6]), f16(p[7])};
        // words of two tokens: [run][pair of the four][half of the chunk], four dims each
#pragma unroll
        for (int n = 0; n < N / 4; ++n) {
            h2 v[4][4];   // [run, pair][dim]
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    uint32_t word;
                    if constexpr (D == 64) word = lane & 1 ? t.vc[i][2 * k + 1] : t.vc[i][2 * k];
                    else word = t.vc[i][(n >> 1) * 4 + 2 * k + (n & 1)];
                    h2 code[4];
                    codes8(word, code);
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        v[2 * i + k][j] = __builtin_elementwise_fma(code[j], as_h2(t.vs[i][k]), as_h2(t.vs[i][2 + k]));
                }
#pragma unroll
            for (int j = 0; j < 4; ++j) o[4 * n + j] = mfma16(join(v[0][j], v[1][j], v[2][j], v[3][j]), w, o[4 * n + j]);
        }
        if (more) {
#pragma unroll
            for (int i = 0; i < 2; ++i) t.values(i, pg[i], slab, in[i], lane);
        }
    }

    // the four waves' sums together
    sum = rows_sum(sum);
    if (lane < 16) {
        top_sh[wave][lane] = top;
        sum_sh[wave][lane] = sum;
    }
    __syncthreads();
    float all = top_sh[0][lane & 15];
#pragma unroll
    for (int i = 1; i < 4; ++i) all = fmaxf(all, top_sh[i][lane & 15]);
    const float f = __builtin_amdgcn_exp2f(top - all);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float* at_row = &part[wave][lane & 15][N * (4 * c + i)];
#pragma unroll
        for (int n = 0; n < N; ++n) at_row[n] = o[n][i] * f;
    }
    if (bad && hi > 0 && lane < 16) sum_sh[wave][lane] = NAN;
    __syncthreads();
    const int r = threadIdx.x >> 4, d = (threadIdx.x & 15) * N;
    if (r >= rows) return;
    float most = top_sh[0][r], total = 0.0f, y[N];
#pragma unroll
    for (int i = 1; i < 4; ++i) most = fmaxf(most, top_sh[i][r]);
#pragma unroll
    for (int i = 0; i < 4; ++i) total += sum_sh[i][r] * __builtin_amdgcn_exp2f(top_sh[i][r] - most);
#pragma unroll
    for (int n = 0; n < N; ++n) y[n] = (part[0][r][d + n] + part[1][r][d + n]) + (part[2][r][d + n] + part[3][r][d + n]);
    const int t_out = (row0 + r) / a.group, h_out = head * a.group + (row0 + r) - t_out * a.group;
    if (a.splits == 1) {
        const float inv = total == 0.0f ? 0.0f : 1.0f / total;
        T v[N];
#pragma unroll
        for (int n = 0; n < N; ++n) v[n] = T(y[n] * inv);
        __builtin_memcpy(static_cast<T*>(a.out) + int64_t(s.first + t_out) * a.out_stride + int64_t(h_out) * D + d, v, sizeof v);
    } else {
        const int64_t i = (int64_t(s.first + t_out) * a.q_heads + h_out) * a.splits + split;
        __builtin_memcpy(a.part + i * D + d, y, sizeof y);
        if (d == 0) {
            a.part_ml[2 * i] = most;
            a.part_ml[2 * i + 1] = total;
        }
    }
}

// The splits' sums together: a workgroup for each row and head, threads of D / 4 and of the splits.
template <class T, int D>
__global__ __launch_bounds__(256) void attend_join_kernel(AttendArgs a) {
    constexpr int L = D / 4, W = 256 / L;   // threads of one split's row, splits at a time
    __shared__ f4 sums[W][L];
    const int64_t row = blockIdx.x;
    const int t = int(row / a.q_heads), h = int(row - int64_t(t) * a.q_heads);
    // rows of no sequence have no parts
    const SeqRows s = seq_rows(a.b, seq_of(a.b, t));
    if (t < s.first || t >= s.first + s.n) return;
    const float* ml = a.part_ml + 2 * row * a.splits;
    float most = kLowest, total = 0.0f;
    for (int i = 0; i < a.splits; ++i) most = fmaxf(most, ml[2 * i]);
    for (int i = 0; i < a.splits; ++i) total += ml[2 * i + 1] * __builtin_amdgcn_exp2f(ml[2 * i] - most);
    const int w = threadIdx.x / L, d = threadIdx.x % L;
    f4 y = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int i = w; i < a.splits; i += W) {
        if (ml[2 * i + 1] == 0.0f) continue;
        y += *reinterpret_cast<const f4*>(a.part + (row * a.splits + i) * D + 4 * d) * __builtin_amdgcn_exp2f(ml[2 * i] - most);
    }
    sums[w][d] = y;
    __syncthreads();
    if (w) return;
#pragma unroll
    for (int i = 1; i < W; ++i) y += sums[i][d];
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
    T v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = T(y[i] * inv);
    __builtin_memcpy(static_cast<T*>(a.out) + int64_t(t) * a.out_stride + int64_t(h) * D + 4 * d, v, sizeof v);
}

template <class T, int D>
hipError_t attend_go(const AttendArgs& a, hipStream_t s, hipEvent_t stop) {
    const uint32_t grid = uint32_t(a.b.n_seqs) * uint32_t(a.tiles) * uint32_t(a.splits) * uint32_t(a.b.kv_heads);
    hipExtLaunchKernelGGL((attend_few_kernel<T, D>), dim3(grid), dim3(256), 0, s, nullptr, a.splits == 1 ? stop : nullptr, 0, a);
    if (a.splits > 1)
        hipExtLaunchKernelGGL((attend_join_kernel<T, D>), dim3(uint32_t(a.b.rows) * uint32_t(a.q_heads)), dim3(256), 0, s, nullptr, stop, 0, a);
    return hipGetLastError();
}
template <class T>
hipError_t attend_type(const AttendArgs& a, hipStream_t s, hipEvent_t stop) {
    switch (a.b.dim) {
    case 64: return attend_go<T, 64>(a, s, stop);
    case 128: return attend_go<T, 128>(a, s, stop);
    case 256: return attend_go<T, 256>(a, s, stop);
    default: return hipErrorInvalidValue;
    }
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
