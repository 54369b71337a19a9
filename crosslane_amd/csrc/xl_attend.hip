// CDNA4 (gfx950) attention over a 4-bit cache.
//
//   out = sum_j p_j v_j / sum_j p_j,   p_j = exp(x_j - m),   x_j = scale * q . k_j
//
// One pass over the tokens: m is a maximum so far, and where a later one passes it by more
// than 2^8 in weight, what was summed is scaled down. Codes of 4 bits become float16 by two
// instructions a pair (bits under an exponent, and that exponent's value off again) and their
// scale and smallest value by one fused multiply-add. Scores, maxima, sums and outputs are
// float32; what is rounded to float16, once each, by at most 2^-11 of itself:
//   - keys and values, since the matrix cores take float16 operands: an eighth of what bfloat16 outputs round away, and as much
//     as float16 ones do, which are so within two to four of their own roundings (rms 3.0e-4 to 7.5e-4 of the outputs' rms over
//     the measured calls, most of it by the keys, where exact operands have 2.1e-4). Keys as two operands each (s * code and what its rounding leaves, m by the sums
//     of q over the groups) gave 3.0e-4 and took 10 to 12 % longer with few rows (637 MB 152 us for 137), and would take
//     twice the LDS and the scores' products with many.
//   - weights, for the second product. Their sum is of the weights before.
// A row before its sequence's first token sees none, and its outputs are zeros. Of every other row the sum of the weights is 1 at
// least, but where its scores pass what float32 holds: then it is 0 or a NaN, and the outputs are NaN.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "xl_act.hpp"
#include "xl_format.hpp"
#include "xl_kv_index.hpp"

namespace xl {
namespace {

// Rows (of a sequence and a kv head) up to which attend_few_kernel takes them, 16 at a time: of 24 sequences with up to 12 rows and
// 9000 tokens, group 4 (48 rows), 59 us for 109 of attend_many_kernel; one sequence of 131072 tokens, 48 rows: 96 for 90,
// 96 rows: 172 for 95; heads of 256, 72 rows: 121 for 229, 192 rows: 231 for 315.
constexpr int few_rows(int dim) { return dim == 256 ? 192 : 64; }

}  // namespace

// Few rows: as many workgroups as the card holds at once (four a CU, two of heads of 256 values) where each has 256 tokens at
// least, or three times as many for an even end where each has 2048; up to 1280 tokens in one piece, which the join's launch
// would cost more than it gives (48 sequences' last 1024 tokens 20 to 30 us, in two or three pieces 26 to 36; one sequence of
// 1024 14.7 in one and in two). Over 77 calls, run with 1 to 128 splits each, 4 % above the best on average and 22 % at most.
// Many rows: the least of the rounds that 512 workgroups at a
// time make (256 of heads of 256), at 0.03 (0.05) us a token that the rows see on average and 5 us a workgroup, and the join's
// bytes at 4 TB/s: over 62 calls of 60 to 2000 rows, run with 1 to 16 splits each, 2 % above the best on average and 18 % at most.
AttendPlan attend_plan(int dim, int kv_heads, int q_heads, int n_seqs, int rows, int max_rows, int64_t max_tokens, int window) {
    AttendPlan p;
    const int64_t group = q_heads / kv_heads, most = max_rows * group;
    const int64_t tokens = window ? std::min(max_tokens, int64_t(window) + max_rows) : max_tokens;
    p.few = most <= few_rows(dim);
    int64_t wgs;
    if (p.few) {
        p.tiles = int((most + 15) / 16);
        wgs = int64_t(n_seqs) * kv_heads * p.tiles;
        const int64_t held = dim < 256 ? 1024 : 512;
        const auto splits = [&](int64_t groups, int64_t least) {
            return std::min(std::max<int64_t>(1, groups / wgs), (tokens + least - 1) / least);
        };
        if (tokens > 1280) p.splits = int(std::min<int64_t>(128, std::max(splits(held, 256), splits(3 * held, 2048))));
    } else {
        p.tiles = int((rows * group >> 7) + n_seqs);   // numbers for them; about half a tile of each sequence has rows
        wgs = int64_t(kv_heads) * p.tiles;
        const int64_t held = dim < 256 ? 512 : 256;
        const double seen = std::max(double(tokens) - 0.5 * max_rows, 0.5 * double(tokens)), us_token = dim < 256 ? 0.03 : 0.05;
        const int64_t real = kv_heads * (((rows * group + 127) >> 7) + (n_seqs - 1) / 2);
        double best = 1e30;
        for (int64_t k = 1; k <= 128 && (k == 1 || (real * k <= 2048 && tokens >= 256 * k)); ++k) {
            const double rounds = double((real * k + held - 1) / held), join = k == 1 ? 0.0 : 4.0 + double(rows) * q_heads * dim * double(k) * 1e-6;
            const double us = rounds * (us_token * seen / double(k) + 5.0) + join;
            if (us < best) {
                best = us;
                p.splits = int(k);
            }
        }
    }
    const int64_t heads = int64_t(rows) * q_heads;
    p.groups = wgs * p.splits;
    if (p.splits > 1) p.groups = std::max(p.groups, p.splits > 16 ? heads : (heads * (dim / 4) + 255) / 256);
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
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

constexpr float kLowest = -3.402823466e38f;   // a maximum before any token (below every score but -inf)
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLazy = 8.0f;                 // weights up to 2^8 before the maximum moves (float16 holds 2^15)

__device__ __forceinline__ h2 as_h2(uint32_t v) { return __builtin_bit_cast(h2, v); }
__device__ __forceinline__ uint32_t as_u32(h2 v) { return __builtin_bit_cast(uint32_t, v); }
__device__ __forceinline__ h2 both(f16 v) { return h2{v, v}; }

// Nibbles 0 and 4, 1 and 5, 2 and 6, 3 and 7 of a word, as pairs of whole numbers in float16: a nibble
// under the exponent of 1024 is 1024 + code, four bits higher under that of 64 it is 64 + code. The masks lie in
// vector registers and the exponents in scalar ones: an instruction takes no two constants, but so it is v_and_or_b32.
struct Codes {
    uint32_t low = 0x000f000fu, high = 0x00f000f0u, e1024 = 0x64006400u, e64 = 0x54005400u;
    __device__ __forceinline__ Codes() { asm("" : "+v"(low), "+v"(high), "+s"(e1024), "+s"(e64)); }
    __device__ __forceinline__ void operator()(uint32_t w, h2 (&c)[4]) const {
        const uint32_t u = w >> 8;
        c[0] = as_h2((w & low) | e1024) - both(f16(1024.0f));
        c[1] = as_h2((w & high) | e64) - both(f16(64.0f));
        c[2] = as_h2((u & low) | e1024) - both(f16(1024.0f));
        c[3] = as_h2((u & high) | e64) - both(f16(64.0f));
    }
};
__device__ __forceinline__ h8 join(h2 a, h2 b, h2 c, h2 d) {
    return __builtin_bit_cast(h8, u4{as_u32(a), as_u32(b), as_u32(c), as_u32(d)});
}
__device__ __forceinline__ f4 mfma16(h8 a, h8 b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

// Whether any lane has a NaN among four pairs of float16 (sums keep one).
__device__ __forceinline__ bool has_nan(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    const h2 v = (as_h2(a) + as_h2(b)) + (as_h2(c) + as_h2(d));
    return __any(v[0] != v[0] || v[1] != v[1]);
}
typedef float f2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ h2 pack(float a, float b) { return __builtin_convertvector(f2{a, b}, h2); }
// Maximum / sum over the four runs of 16 lanes, in every lane.
__device__ __forceinline__ float rows_max(float v) {
    v = fmaxf(v, __shfl_xor(v, 16));
    return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float rows_sum(float v) {
    v += __shfl_xor(v, 16);
    return v + __shfl_xor(v, 32);
}
// Scores through softcap * tanh(score / softcap), of a row's products x: tanh y = 2 / (1 + exp(-2 y)) - 1. A row's scores may all be off
// by the same, so the -1 is left out: 1 / (1 + exp(-2 y)) of each, and twice softcap (times log2(e)) as the row's factor. What this
// rounds is 2^-23 of softcap, so the host takes softcap up to 2^14 only (0.003 of a score). (Written with the -1: the largest prefill
// with a softcap 837 instead of 760 us; 710 to 760 by card, 580 to 660 without a cap: 8,350 more vector instructions a wave on 19,440.)
struct Cap {
    float in, out;   // (a factor that would be infinite makes 0 of no product NaN)
    __device__ __forceinline__ Cap(float softcap, float up) : in(fmaxf(-2.0f * kLog2e / softcap * up, -3.4e38f)), out(2.0f * softcap * kLog2e) {}
    __device__ __forceinline__ float operator()(float x) const { return __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(x * in) + 1.0f); }
};

// A lane's part of a row of q in float16 (K chunks of eight values), which `most` joins with the row's other lanes; a scale
// below 0 turns it, so that the largest product is the largest score. A bfloat16 row is taken times a power of two that
// brings its largest value to 1..2, so that float16 holds all its bits, down to 2^-25 of that value. A row with a value that is
// not finite is all NaN. Returns what takes its products to scores, times log2(e) unless a cap follows: above 0, so that
// -inf stays hidden.
template <class T, int K, class F>
__device__ __forceinline__ float take_q(const AttendArgs& a, const T* p, int stride, h8 (&q)[K], F&& most) {
    typedef uint16_t s2 __attribute__((ext_vector_type(2)));
    u4 w[K];
#pragma unroll
    for (int k = 0; k < K; ++k) __builtin_memcpy(&w[k], p + k * stride, 16);
    s2 m = {0, 0};   // magnitudes order as their bits
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) m = __builtin_elementwise_max(m, __builtin_bit_cast(s2, w[k][i] & 0x7fff7fffu));
    const uint32_t top = most(max(uint32_t(m[0]), uint32_t(m[1])));
    constexpr bool BF = __is_same(T, bf16);
    const bool bad = top >= (BF ? 0x7f80u : 0x7c00u);
    const int e = BF ? (top < 0x80u ? -126 : int(top >> 7) - 127) : 0;   // (subnormal rows: as the smallest normal ones)
    const float sign = bad ? NAN : a.scale < 0.0f ? -1.0f : 1.0f;
    if constexpr (BF) {
        const float f = __builtin_amdgcn_ldexpf(sign, -e);
#pragma unroll
        for (int k = 0; k < K; ++k) {
            h2 v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = pack(__uint_as_float(w[k][i] << 16) * f, __uint_as_float(w[k][i] & 0xffff0000u) * f);
            q[k] = join(v[0], v[1], v[2], v[3]);
        }
    } else {
        const h2 f = both(f16(sign));
#pragma unroll
        for (int k = 0; k < K; ++k) q[k] = join(as_h2(w[k][0]) * f, as_h2(w[k][1]) * f, as_h2(w[k][2]) * f, as_h2(w[k][3]) * f);
    }
    return fmaxf(__builtin_amdgcn_ldexpf(fabsf(a.scale) * (a.softcap > 0.0f ? 1.0f : kLog2e), e), 1.17549435e-38f);
}

// What a lane loads of a tile of 32 tokens (two runs of 16), for keys as the first operand of the scores
// (token lane % 16 of each run, the eight dims 32g + 8c with c = lane / 16 of every group g), and for values as
// the first operand of the outputs (dims D / 16 * (lane % 16) on, the four tokens 4c of each run). An address is a
// run's place, the same for the wave, and an offset of the lane's that stays. ONCE: nobody else reads these bytes.
template <int D, bool ONCE>
struct TileLoads {
    static constexpr int G = D / 32;
    uint32_t kc[2][G], ks[2][G], vc[2][D >= 128 ? D / 32 : 4], vs[2][4];
    uint32_t kc_at, ks_at, vc_at, vs_at;
    template <int N>
    static __device__ __forceinline__ void load(const uint8_t* p, uint32_t (&w)[N]) {
        if constexpr (ONCE) {
            typedef uint32_t V __attribute__((ext_vector_type(N)));
            const V v = __builtin_nontemporal_load(reinterpret_cast<const V*>(p));
            __builtin_memcpy(w, &v, sizeof v);
        } else {
            __builtin_memcpy(w, __builtin_assume_aligned(p, N >= 4 ? 16 : 4 * N), 4 * N);
        }
    }
    __device__ __forceinline__ explicit TileLoads(int lane) {
        const int tok = lane & 15, c = lane >> 4, chunk = D >= 128 ? tok * (D / 128) : tok >> 1;
        kc_at = 4 * (tok * (D / 8) + c * G);
        ks_at = 4 * tok * G;
        vc_at = 2 * (c * D + chunk * 8);
        vs_at = 16 * (c * G + chunk / 4);
    }
    __device__ __forceinline__ void keys(int i, const uint8_t* slab, const Slab<D>& s, int run) {
        load(slab + 8 * D * run + kc_at, kc[i]);
        load(slab + s.k_scales() + 64 * G * run + ks_at, ks[i]);
    }
    __device__ __forceinline__ void values(int i, const uint8_t* slab, const Slab<D>& s, int run) {
        load(slab + s.v_codes() + 8 * D * run + vc_at, vc[i]);
        load(slab + s.v_scales() + 64 * G * run + vs_at, vs[i]);
    }
};

// A load at an address that is the same for the wave, of memory that the kernel does not write: by the scalar unit.
__device__ __forceinline__ int scalar_load(const int32_t* p) {
    return *(const __attribute__((address_space(4))) int32_t*)(reinterpret_cast<uintptr_t>(p));
}

// Few rows (of one sequence and kv head: its tokens' rows, each with `group` heads): a workgroup has 16 of them and
// one of `splits` parts of the tokens, its four waves every fourth tile of 32.
//
// Bound by the cache's bytes where each is read once (4.8 to 5.0 TB/s of 64 sequences of up to 16384 tokens and of one
// sequence of 131072, as a copy), else by the conversion, which each 16 rows do anew. A wave makes score^T = K q^T and out^T = V^T p^T with
// v_mfma_f32_16x16x32_f16: keys and values go from memory to registers and from there into the matrix cores as the
// first operand, with no LDS and no exchange between lanes; the scores come out in the lanes (row lane % 16, tokens
// 4 (lane / 16) ..+3 of each run) where the second product wants its weights, since the order of tokens
// within its sum is free. Loads of the next tile follow the last use of this one's registers.
template <class T, int D, bool ONCE>
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
    const int per = max(8, ((tiles + a.splits - 1) / a.splits + 3) & ~3);
    const int begin = tile0 + split * per + wave, end = tile0 + min(tiles, (split + 1) * per);

    const Slab<D> slab(b.page);
    const uint8_t* base = b.pages + int64_t(head) * slab.bytes();
    const int first_run = lo_all >> 4, last_run = (hi_all - 1) >> 4;
    TileLoads<D, ONCE> t(lane);
    const Codes codes;
    // A tile's pages, by the table's entries, which are read a tile before they are used. A run before the first token that a row
    // sees, or behind the last, is the first or last run with such a token (other pages may be gone); where an entry is no page,
    // the first page: such tokens are hidden.
    const int32_t* row_of_table = b.table + int64_t(seq) * b.table_stride;
    int id[2], in[2];
    const auto look = [&](int tl, int first = INT32_MIN) {   // (the first tile alone has a run before the first token)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t run = uint32_t(min(max(2 * tl + i, first), last_run));
            const uint32_t col = b.page_inv ? __umulhi(run, b.page_inv) : run;
            in[i] = int(run - col * uint32_t(b.page >> 4));
            id[i] = scalar_load(row_of_table + col);
        }
    };
    const uint8_t* pg[2];
    int run[2];
    bool ok[2];
    const auto turn_to = [&] {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            ok[i] = uint32_t(id[i]) < uint32_t(b.n_pages);
            pg[i] = base + (ok[i] ? int64_t(id[i]) * b.page_stride : 0);
            run[i] = in[i];
        }
    };
    if (begin < end) {
        look(begin, first_run);
        turn_to();
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            t.keys(i, pg[i], slab, run[i]);
            t.values(i, pg[i], slab, run[i]);
        }
        if (begin + 4 < end) look(begin + 4);
        if (32 * begin < lo_all) {   // values before the first token that a row sees
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (32 * begin + 16 * (j >> 2) + 4 * c + (j & 3) < lo_all) {
                    t.vs[j >> 2][(j & 3) >> 1] &= j & 1 ? 0x0000ffffu : 0xffff0000u;
                    t.vs[j >> 2][2 + ((j & 3) >> 1)] &= j & 1 ? 0x0000ffffu : 0xffff0000u;
                }
        }
    }

    // q: the second operand, row lane % 16, dims 32g + 8c ..+7
    h8 q[G];
    const float up = take_q(a, static_cast<const T*>(a.q) + int64_t(s.first + row_t) * a.q_stride + int64_t(row_h) * D + 8 * c, 32, q,
                            [](uint32_t v) {
                                v = max(v, uint32_t(__shfl_xor(int(v), 16)));
                                return max(v, uint32_t(__shfl_xor(int(v), 32)));
                            });
    const Cap cap(a.softcap, up);
    const float upx = a.softcap > 0.0f ? cap.out : up;

    float top = kLowest, sum = 0.0f;
    f4 o[N] = {};
    for (int tl = begin; tl < end; tl += 4) {
        const bool more = tl + 4 < end, ok0 = ok[0], ok1 = ok[1];
        if (more) {
            turn_to();
            if (tl + 8 < end) look(tl + 8);
        }
        float x[8];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            f4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int g = 0; g < G; ++g) {
                const h2 sm = as_h2(t.ks[i][g]), step = both(sm[0]), small = both(sm[1]);
                h2 k[4];
                codes(t.kc[i][g], k);
#pragma unroll
                for (int j = 0; j < 4; ++j) k[j] = __builtin_elementwise_fma(k[j], step, small);
                acc = mfma16(join(k[0], k[1], k[2], k[3]), q[g], acc);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) x[4 * i + j] = acc[j];
        }
        if (more) {
#pragma unroll
            for (int i = 0; i < 2; ++i) t.keys(i, pg[i], slab, run[i]);
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
                    t.vs[j >> 2][(j & 3) >> 1] &= j & 1 ? 0x0000ffffu : 0xffff0000u;
                    t.vs[j >> 2][2 + ((j & 3) >> 1)] &= j & 1 ? 0x0000ffffu : 0xffff0000u;
                }
            }
            if (lane == 0 && !(ok0 && ok1)) atomicOr(b.err, kDevErrBatch);
        }
        float m = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7]))) * upx;
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
            p[j] = __builtin_amdgcn_exp2f(fmaf(x[j], upx, -top));
            sum += p[j];
        }
        // a token held as NaN: its values as 0, and the rows that see it NaN by their sum
        if (has_nan(t.vs[0][0], t.vs[0][1], t.vs[1][0], t.vs[1][1])) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                uint32_t& w0 = t.vs[j >> 2][(j & 3) >> 1];
                uint32_t& w1 = t.vs[j >> 2][2 + ((j & 3) >> 1)];
                const uint32_t e = (j & 1 ? w0 >> 16 : w0) & 0x7fffu;
                if (e >= 0x7c00u) {
                    w0 &= j & 1 ? 0x0000ffffu : 0xffff0000u;
                    w1 &= j & 1 ? 0x0000ffffu : 0xffff0000u;
                    if (x[j] != -INFINITY) sum = NAN;
                }
            }
        }
        const h8 w = join(pack(p[0], p[1]), pack(p[2], p[3]), pack(p[4], p[5]), pack(p[6], p[7]));
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
                    codes(word, code);
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        v[2 * i + k][j] = __builtin_elementwise_fma(code[j], as_h2(t.vs[i][k]), as_h2(t.vs[i][2 + k]));
                }
#pragma unroll
            for (int j = 0; j < 4; ++j) o[4 * n + j] = mfma16(join(v[0][j], v[1][j], v[2][j], v[3][j]), w, o[4 * n + j]);
        }
        if (more) {
#pragma unroll
            for (int i = 0; i < 2; ++i) t.values(i, pg[i], slab, run[i]);
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
        const float inv = before + t_out < 0 ? 0.0f : 1.0f / total;
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

// Many rows: a workgroup has 128 (of one sequence and kv head), its four waves 32 each, and one of `splits` parts
// of the tokens, TT at a time.
//
// Bound by matrix and vector instructions alike: a tile's 16 + 16 products of v_mfma_f32_32x32x16_f16 take a wave 1024 cycles, and
// the softmax of its 32 scores a lane with a quarter of the tile's codes made float16 about as many. So the workgroup makes them
// once for all its rows, into LDS (keys as rows of dims, values as rows of tokens), scores stay in the lanes that need them as weights,
// as above (values' tokens lie in LDS in the order in which the scores come out), and both kinds of instructions go side by side:
// a tile's exponentials between the next tile's scores, and the codes of later tiles between its values' products, a slice to
// a product, in an order that the compiler is kept from changing (8192 tokens of 32 heads of 128: 607 us for 621 of one kind after
// the other; now 580 to 660 by card). That is 830 to 950 TFLOP/s, 70 to 80 % of what the library's products of float16 reach.
// 128 rows and two workgroups a CU: 256 rows in eight waves, one workgroup a CU, took as long (576 for 578 us).
template <int D>
struct Many {
    static constexpr int TT = D == 256 ? 32 : 64;   // tokens of a tile
    static constexpr int G = D / 32, C = D / 8, KS = D / 16, NT = D / 32, MT = TT / 32;
    // What a thread makes of a tile: KW words of one token's keys; of values the words of VP of the two pairs of four tokens, eight dims.
    static constexpr int KW = TT * C / 256, VP = TT * C / 512;
    // Rows in LDS are 16 bytes longer than their values, so that eight lanes' 16 bytes of eight rows lie in banks of their own. A
    // value's row is (dim % 8) * C + dim / 8: the lanes that write, of chunks of eight dims, have neighbouring rows then.
    static constexpr int KROW = D + 8, VROW = TT + 8;
};
typedef float f16x __attribute__((ext_vector_type(16)));

template <class T, int D, bool CAP>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void attend_many_kernel(AttendArgs a) {
    using M = Many<D>;
    constexpr int TT = M::TT, G = M::G, C = M::C, KW = M::KW, VP = M::VP, KROW = M::KROW, VROW = M::VROW;
    __shared__ __attribute__((aligned(16))) f16 ksh[2][TT * KROW];
    __shared__ __attribute__((aligned(16))) f16 vsh[2][D * VROW];
    const KvBatch& b = a.b;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), c = lane >> 5;
    // Sequence q's tiles are numbered from starts[q] * group / 128 + q on: at least as many numbers as it has tiles. The last ones,
    // which see the most tokens, go first.
    uint32_t at = blockIdx.x;
    const int head = at % b.kv_heads;
    at /= b.kv_heads;
    const int split = at % a.splits;
    const int number = a.tiles - 1 - int(at / a.splits);
    const auto first_number = [&](int q) { return int(int64_t(scalar_load(b.starts + q)) * a.group >> 7) + q; };
    int seq = 0;
    for (int hi = b.n_seqs; hi - seq > 1;) {
        const int mid = (seq + hi) >> 1;
        if (first_number(mid) <= number) seq = mid;
        else hi = mid;
    }
    if (blockIdx.x == 0)
        for (int i = tid; i < b.n_seqs; i += 256)
            if (seq_rows(b, i).bad) atomicOr(b.err, kDevErrBatch);
    const SeqRows s = seq_rows(b, seq);
    const int row0 = 128 * (number - first_number(seq)), rows = min(128, s.n * a.group - row0);
    if (row0 < 0 || rows <= 0) return;
    const int before = s.len - s.n;
    const auto sees = [&](int row) { return before + row / a.group + 1; };   // tokens up to a row's own
    const auto from = [&](int upto) { return a.window ? max(0, upto - a.window) : 0; };
    // this lane's row, and the tokens that it sees: lo ..hi - 1; the same for the wave's first and last row, and the workgroup's
    const int row = row0 + min(32 * wave + (lane & 31), rows - 1), row_t = row / a.group;
    const int row_h = head * a.group + row - row_t * a.group;
    const int hi = before + row_t + 1, lo = from(hi);
    const int hi_least = sees(row0 + min(32 * wave, rows - 1)), lo_most = from(sees(row0 + min(32 * wave + 31, rows - 1)));
    const int hi_all = sees(row0 + rows - 1), lo_all = from(sees(row0));
    const int tile0 = lo_all / TT, tiles = hi_all > lo_all ? (hi_all + TT - 1) / TT - tile0 : 0;
    const int per = max(256 / TT, (tiles + a.splits - 1) / a.splits);
    const int begin = tile0 + split * per, end = tile0 + min(tiles, (split + 1) * per);

    // This thread's part of a tile: words of one token's keys, and eight dims of four (or two) tokens' values. A wave's lie in one run
    // of 16 tokens, whose page is looked up a tile before it is used; a run before the first token that a row sees, or behind the
    // last, is the first or last run with such a token (other pages may be gone), an entry that is no page the first page. Keys are
    // loaded a tile before the values of the same tokens.
    const Slab<D> slab(b.page);
    const Codes codes;
    const uint8_t* base = b.pages + int64_t(head) * slab.bytes();
    const int32_t* row_of_table = b.table + int64_t(seq) * b.table_stride;
    const int k_tok = tid / (C / KW), k_sub = tid % (C / KW);
    const int v_quad = tid / (2 / VP * C), v_chunk = tid / (2 / VP) % C, v_pair = VP == 1 ? tid & 1 : 0;
    const uint32_t kc_at = 4 * ((k_tok & 15) * C + KW * k_sub);
    const uint32_t ks_at = slab.k_scales() + 4 * ((k_tok & 15) * G + KW * k_sub % G);
    const uint32_t kv_at = slab.v_scales() + 2 * ((k_tok >> 2 & 3) * 8 * G + (k_tok & 3));   // the scale of the same token's values
    const uint32_t vc_at = slab.v_codes() + 2 * ((v_quad & 3) * D + v_chunk * 8) + 8 * v_pair;
    const uint32_t vs_at = slab.v_scales() + 16 * ((v_quad & 3) * G + v_chunk / 4) + 4 * v_pair;
    const int first_run = lo_all >> 4, last_run = (hi_all - 1) >> 4;
    struct Page {
        int id, in;
    };
    struct Run {   // where a run's codes begin, and its scales, both without their parts' offsets
        const uint8_t *code, *scale;
        bool ok;
    };
    const auto look = [&](int tl, int first = INT32_MIN) {   // (the first tile alone has runs before the first token)
        const uint32_t run = uint32_t(min(max(TT == 64 ? 4 * tl + wave : 2 * tl + (wave >> 1), first), last_run));
        const uint32_t col = b.page_inv ? __umulhi(run, b.page_inv) : run;
        return Page{scalar_load(row_of_table + col), int(run - col * uint32_t(b.page >> 4))};
    };
    const auto run_of = [&](const Page& p) {
        const bool ok = uint32_t(p.id) < uint32_t(b.n_pages);
        const uint8_t* at = base + (ok ? int64_t(p.id) * b.page_stride : 0);
        return Run{at + 8 * D * p.in, at + 64 * G * p.in, ok};
    };
    struct RawKeys {
        uint32_t code[KW], scale[KW < G ? KW : G];
        f16 of_value;
        bool ok;
    };
    struct RawValues {
        uint32_t code[2 * VP], step[VP], small[VP];   // [pair][half]; [pair]
        bool ok;
    };
    const auto fetch_keys = [&](const Run& at, RawKeys& r) {
        __builtin_memcpy(r.code, __builtin_assume_aligned(at.code + kc_at, sizeof r.code), sizeof r.code);
        __builtin_memcpy(r.scale, __builtin_assume_aligned(at.scale + ks_at, sizeof r.scale), sizeof r.scale);
        r.of_value = *reinterpret_cast<const f16*>(at.scale + kv_at);
        r.ok = at.ok;
    };
    const auto fetch_values = [&](const Run& at, RawValues& r) {
        __builtin_memcpy(r.code, __builtin_assume_aligned(at.code + vc_at, sizeof r.code), sizeof r.code);
        if constexpr (VP == 2) {
            uint32_t w[4];
            __builtin_memcpy(w, __builtin_assume_aligned(at.scale + vs_at, 16), 16);
            r.step[0] = w[0], r.step[VP - 1] = w[1], r.small[0] = w[2], r.small[VP - 1] = w[3];
        } else {
            r.step[0] = *reinterpret_cast<const uint32_t*>(at.scale + vs_at);
            r.small[0] = *reinterpret_cast<const uint32_t*>(at.scale + vs_at + 8);
        }
        r.ok = at.ok;
    };
    // word i of the thread's keys is c * G + g of its token: unit 4g + c of eight dims
    f16* const k_put = &ksh[0][k_tok * KROW + 8 * (D == 256 ? 16 * (k_sub & 1) + (k_sub >> 1) : k_sub)];
    f16* const v_put = &vsh[0][v_chunk * VROW + 16 * (v_quad >> 2) + 8 * (v_quad & 1) + 4 * (v_quad >> 1 & 1) + 2 * v_pair];
    // The codes to float16, in slices that go between products: of keys two for each word; of values, for each half of the eight dims,
    // the codes of each pair of tokens, then as many slices of their dims. Where a token's values are held as NaN, so are its
    // keys here, which the scores carry to the rows that see it; the values become numbers (maxima leave a NaN), since a
    // weight of 0 makes no 0 of a NaN.
    constexpr int KSLICES = 2 * KW, VSLICES = 4 * VP;
    h2 codes_of[VP][4];
    const auto stage_keys = [&](const RawKeys& r, int buf, int slice) {
        const int i = slice / 2;
        if (slice % 2 == 0) {
            codes(r.code[i], codes_of[0]);
        } else {
            h2 sm = as_h2(r.scale[i % (KW < G ? KW : G)]);
            if (i == 0) sm[1] = __builtin_elementwise_fma(r.of_value, f16(0.0f), sm[1]);
            h2 k[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) k[j] = __builtin_elementwise_fma(codes_of[0][j], both(sm[0]), both(sm[1]));
            *reinterpret_cast<h8*>(k_put + buf * (TT * KROW) + 32 * i) = join(k[0], k[1], k[2], k[3]);
        }
    };
    const auto stage_values = [&](const RawValues& r, int buf, int slice) {
        const int h = slice / (2 * VP), k = slice % (2 * VP);
        if (k < VP) {
            codes(r.code[2 * k + h], codes_of[k]);
        } else {
#pragma unroll
            for (int j = (k - VP) * (4 / VP); j < (k - VP + 1) * (4 / VP); ++j) {
                f16* at = v_put + buf * (D * VROW) + (4 * h + j) * C * VROW;
                uint32_t v[VP];
#pragma unroll
                for (int i = 0; i < VP; ++i) v[i] = as_u32(__builtin_elementwise_fma(codes_of[i][j], as_h2(r.step[i]), as_h2(r.small[i])));
                __builtin_memcpy(__builtin_assume_aligned(at, sizeof v), v, sizeof v);
            }
        }
    };
    // Values that no row sees are 0, and those of a page that is none (whose keys are 0 too); none is NaN.
    const auto check_values = [&](RawValues& r, int tl) {
#pragma unroll
        for (int i = 0; i < VP; ++i) {
            r.step[i] = as_u32(__builtin_elementwise_max(as_h2(r.step[i]), both(f16(0.0f))));
            r.small[i] = as_u32(__builtin_elementwise_max(as_h2(r.small[i]), both(f16(-65504.0f))));
        }
        if (TT * (tl + 1) > hi_all || !r.ok) {
#pragma unroll
            for (int i = 0; i < VP; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j)
                    if (TT * tl + 4 * v_quad + 2 * (v_pair + i) + j >= hi_all || !r.ok) {
                        r.step[i] &= j ? 0x0000ffffu : 0xffff0000u;
                        r.small[i] &= j ? 0x0000ffffu : 0xffff0000u;
                    }
            if (!r.ok && TT * tl + 4 * v_quad < hi_all) atomicOr(b.err, kDevErrBatch);
        }
    };
    const auto check_keys = [&](RawKeys& r) {
        if (!r.ok) {
#pragma unroll
            for (int i = 0; i < (KW < G ? KW : G); ++i) r.scale[i] = 0;
            r.of_value = f16(0.0f);
        }
    };

    // q: the second operand, row lane % 32, dims 16k + 8c ..+7
    h8 q[M::KS];
    const float up = take_q(a, static_cast<const T*>(a.q) + int64_t(s.first + row_t) * a.q_stride + int64_t(row_h) * D + 8 * c, 16, q,
                            [](uint32_t v) { return max(v, uint32_t(__shfl_xor(int(v), 32))); });
    const Cap cap(a.softcap, up);
    const float upx = CAP ? cap.out : up;

    float top = kLowest, sum = 0.0f;
    f16x o[M::NT] = {};
    const f16* const k_get = &ksh[0][(lane & 31) * KROW + 8 * c];
    const f16* const v_get = &vsh[0][(lane & 31) * VROW + 8 * c];
    constexpr int AHEAD = 2;                                  // operands read from LDS before their products
    constexpr int P1 = M::MT * M::KS, P2 = M::NT * TT / 16;   // products of the scores, and of the values
    const auto key = [&](int buf, int i) {
        return *reinterpret_cast<const h8*>(k_get + buf * (TT * KROW) + 32 * (i % M::MT) * KROW + 16 * (i / M::MT));
    };
    const auto value = [&](int buf, int i) {
        return *reinterpret_cast<const h8*>(v_get + buf * (D * VROW) + 32 * (i % M::NT) * VROW + 16 * (i / M::NT));
    };
    // Products of the scores x with tile `buf`'s keys, and beside(i) between them; nothing moves from one to the next.
    const auto score = [&](f16x (&x)[M::MT], int buf, auto&& beside) {
        h8 k[AHEAD + 1];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) k[i] = key(buf, i);
#pragma unroll
        for (int i = 0; i < P1; ++i) {
            if (i + AHEAD < P1) k[(i + AHEAD) % (AHEAD + 1)] = key(buf, i + AHEAD);
            const f16x before = i < M::MT ? f16x{} : x[i % M::MT];
            x[i % M::MT] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k[i % (AHEAD + 1)], q[i / M::MT], before, 0, 0, 0);
            beside(i);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    // A part of new scores: capped where there is a cap, and the largest so far.
    float most;
    const auto look_over = [&](f16x (&x)[M::MT], bool fresh, int begin_at, int end_at) {
#pragma unroll
        for (int i = begin_at; i < end_at; ++i) {
            if (CAP && fresh) x[i / 16][i % 16] = cap(x[i / 16][i % 16]);
            most = fmaxf(most, x[i / 16][i % 16]);
        }
    };
    constexpr int S = 16 * M::MT;   // scores of a lane
    f16x x0[M::MT], x1[M::MT];
    RawKeys k_raw;
    RawValues v_raw;
    Page page{};    // of the keys to load the next but one time
    Run k_run{}, v_run{};   // of the keys and values to load next
    // One tile, whose scores are in x and their largest in `most`: their exponentials beside the next tile's products (to y); then the
    // values' products beside the codes of the keys of the tile after the next and of the next one's values, loaded a tile before.
    // Behind the last tile that is work on tokens that are there, not used.
    const auto tile = [&](f16x (&x)[M::MT], f16x (&y)[M::MT], int tl) {
        const int buf = (tl - begin) & 1;
        // The stores of the tile before are done before the barrier hands them over. It is stated here: the wait of __syncthreads() is
        // left out by the compiler round the loop, whose entry has nothing outstanding.
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __syncthreads();
        if (TT * tl < lo_most || TT * (tl + 1) > hi_least) {   // tokens that some rows do not see
#pragma unroll
            for (int i = 0; i < S; ++i) {
                const int tok = TT * tl + 32 * (i / 16) + 8 * (i % 16 >> 2) + 4 * c + (i & 3);
                if (tok < lo || tok >= hi) x[i / 16][i % 16] = -INFINITY;
            }
            most = kLowest;
            look_over(x, false, 0, S);
        }
        most *= upx;
        if (__any(most > top + kLazy)) {
            const float m = fmaxf(fmaxf(most, __shfl_xor(most, 32)), top);
            const float f = __builtin_amdgcn_exp2f(top - m);
            top = m;
            sum *= f;
#pragma unroll
            for (int n = 0; n < M::NT; ++n) o[n] *= f;
        }
        h2 w[S / 2];
        score(y, buf ^ 1, [&](int i) {
#pragma unroll
            for (int j = i * S / P1; j < (i + 1) * S / P1; ++j) {
                const float p = __builtin_amdgcn_exp2f(fmaf(x[j / 16][j % 16], upx, -top));
                sum += p;
                if (j & 1) w[j / 2] = pack(x[j / 16][j % 16 - 1], p);
                else x[j / 16][j % 16] = p;
                if (j & 1) asm volatile("" : "+v"(w[j / 2]), "+v"(sum));   // (keeps the exponentials in their place)
            }
        });
        check_keys(k_raw);
        check_values(v_raw, tl + 1);
        most = kLowest;
        h8 v[AHEAD + 1];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) v[i] = value(buf, i);
#pragma unroll
        for (int i = 0; i < P2; ++i) {
            if (i + AHEAD < P2) v[(i + AHEAD) % (AHEAD + 1)] = value(buf, i + AHEAD);
            const int k = 4 * (i / M::NT);
            o[i % M::NT] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v[i % (AHEAD + 1)], join(w[k], w[k + 1], w[k + 2], w[k + 3]), o[i % M::NT], 0, 0, 0);
            if (i < KSLICES) stage_keys(k_raw, buf, i);
            else stage_values(v_raw, buf ^ 1, i - KSLICES);
            if (i == KSLICES) fetch_keys(k_run, k_raw);
            look_over(y, true, i * S / P2, (i + 1) * S / P2);
            __builtin_amdgcn_sched_barrier(0);
        }
        static_assert(VSLICES + KSLICES == P2);
        fetch_values(v_run, v_raw);
        v_run = k_run;
        k_run = run_of(page);
        page = look(tl + 5);
    };
    if (begin < end) {
        RawKeys next;
        const Run r0 = run_of(look(begin, first_run)), r1 = run_of(look(begin + 1));
        fetch_keys(r0, k_raw);
        fetch_values(r0, v_raw);
        fetch_keys(r1, next);
        v_run = run_of(look(begin + 2));
        k_run = run_of(look(begin + 3));
        page = look(begin + 4);
        check_keys(k_raw);
        check_values(v_raw, begin);
        if (TT * begin < lo_all) {   // values before the first token that a row sees
#pragma unroll
            for (int i = 0; i < VP; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j)
                    if (TT * begin + 4 * v_quad + 2 * (v_pair + i) + j < lo_all) {
                        v_raw.step[i] &= j ? 0x0000ffffu : 0xffff0000u;
                        v_raw.small[i] &= j ? 0x0000ffffu : 0xffff0000u;
                    }
        }
#pragma unroll
        for (int i = 0; i < KSLICES; ++i) stage_keys(k_raw, 0, i);
#pragma unroll
        for (int i = 0; i < VSLICES; ++i) stage_values(v_raw, 0, i);
        fetch_keys(v_run, k_raw);
        fetch_values(r1, v_raw);
        check_keys(next);
#pragma unroll
        for (int i = 0; i < KSLICES; ++i) stage_keys(next, 1, i);
        __syncthreads();
        score(x0, 0, [](int) {});
        most = kLowest;
        look_over(x0, true, 0, S);
    }
    for (int tl = begin; tl < end; tl += 2) {
        tile(x0, x1, tl);
        if (tl + 1 < end) tile(x1, x0, tl + 1);
    }

    sum += __shfl_xor(sum, 32);
    if (32 * wave + (lane & 31) >= rows) return;
    // the lane has chunks 8u + 4c + i of its row, whose eight dims lie in as many registers (of row j * C + chunk of the products)
    const int64_t out_row = int64_t(s.first + row_t), part = (out_row * a.q_heads + row_h) * a.splits + split;
    const float inv = a.splits > 1 ? 1.0f : hi <= 0 ? 0.0f : 1.0f / sum;
#pragma unroll
    for (int u = 0; u < C / 8; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float y[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int r = j * C + 8 * u;
                y[j] = o[r >> 5][4 * ((r & 31) >> 3) + i] * inv;
            }
            const int d = 8 * (8 * u + 4 * c + i);
            if (a.splits == 1) store8(static_cast<T*>(a.out) + out_row * a.out_stride + int64_t(row_h) * D + d, 8, y);
            else store8(a.part + part * D + d, 8, y);
        }
    if (a.splits > 1 && c == 0) {
        a.part_ml[2 * part] = top;
        a.part_ml[2 * part + 1] = sum;
    }
}

// The splits' sums together, few splits: a thread has four dims of a row and head, and all of its splits.
template <class T, int D>
__global__ __launch_bounds__(256) void attend_join_few_kernel(AttendArgs a) {
    constexpr int L = D / 4;
    const int64_t row = (int64_t(blockIdx.x) * 256 + threadIdx.x) / L;
    const int d = 4 * (threadIdx.x % L), t = int(row / a.q_heads), h = int(row - int64_t(t) * a.q_heads);
    if (t >= a.b.rows) return;
    const SeqRows s = seq_rows(a.b, seq_of(a.b, t));
    if (t < s.first || t >= s.first + s.n) return;   // rows of no sequence have no parts
    const f2* ml = reinterpret_cast<const f2*>(a.part_ml) + row * a.splits;
    const float* p = a.part + row * a.splits * D + d;
    float most = kLowest, total = 0.0f;
    for (int i = 0; i < a.splits; ++i) most = fmaxf(most, ml[i][0]);
    f4 y = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
    for (int i = 0; i < a.splits; ++i) {
        const float f = __builtin_amdgcn_exp2f(ml[i][0] - most);
        total += ml[i][1] * f;
        y += *reinterpret_cast<const f4*>(p + i * D) * f;
    }
    const float inv = s.len - s.n + t - s.first < 0 ? 0.0f : 1.0f / total;
    T v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = T(y[i] * inv);
    __builtin_memcpy(static_cast<T*>(a.out) + int64_t(t) * a.out_stride + int64_t(h) * D + d, v, sizeof v);
}

// ... many splits: a workgroup for each row and head, 1024 / D splits at a time. Its waves have the splits' maxima and sums in
// their lanes (two each: at most 128), and the weights from there.
template <class T, int D>
__global__ __launch_bounds__(256) void attend_join_kernel(AttendArgs a) {
    constexpr int L = D / 4, P = 64 / L;   // lanes of one split's row, splits at a time in a wave
    __shared__ f4 sums[4][L];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t row = blockIdx.x;
    const int t = int(row / a.q_heads), h = int(row - int64_t(t) * a.q_heads);
    const SeqRows s = seq_rows(a.b, seq_of(a.b, t));
    if (t < s.first || t >= s.first + s.n) return;   // rows of no sequence have no parts
    const f2* ml = reinterpret_cast<const f2*>(a.part_ml) + row * a.splits;
    const f2 none = {kLowest, 0.0f};
    const f2 u = lane < a.splits ? ml[lane] : none, v = lane + 64 < a.splits ? ml[lane + 64] : none;
    float most = fmaxf(u[0], v[0]);
#pragma unroll
    for (int i = 32; i; i >>= 1) most = fmaxf(most, __shfl_xor(most, i));
    const float fu = __builtin_amdgcn_exp2f(u[0] - most), fv = __builtin_amdgcn_exp2f(v[0] - most);
    float total = u[1] * fu + v[1] * fv;
#pragma unroll
    for (int i = 32; i; i >>= 1) total += __shfl_xor(total, i);
    const float* p = a.part + row * a.splits * D + 4 * (lane % L);
    f4 y = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int k = wave * P; k < a.splits; k += 32 * P) {   // eight loads on their way
        f4 x[8];
        float f[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int i = k + j * 4 * P + lane / L, in = min(i, a.splits - 1);
            x[j] = *reinterpret_cast<const f4*>(p + int64_t(in) * D);
            const float f0 = __shfl(fu, in & 63), f1 = __shfl(fv, in & 63);
            f[j] = i >= a.splits ? 0.0f : in < 64 ? f0 : f1;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) y += x[j] * f[j];
    }
#pragma unroll
    for (int i = L; i < 64; i <<= 1)
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] += __shfl_xor(y[j], i);
    if (lane < L) sums[wave][lane] = y;
    __syncthreads();
    if (threadIdx.x >= L) return;
#pragma unroll
    for (int i = 1; i < 4; ++i) y += sums[i][lane];
    const float inv = s.len - s.n + t - s.first < 0 ? 0.0f : 1.0f / total;
    T o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = T(y[i] * inv);
    __builtin_memcpy(static_cast<T*>(a.out) + int64_t(t) * a.out_stride + int64_t(h) * D + 4 * lane, o, sizeof o);
}

template <class T, int D>
hipError_t attend_go(const AttendArgs& a, hipStream_t s) {
    const uint32_t grid = uint32_t(a.few ? a.b.n_seqs : 1) * uint32_t(a.tiles) * uint32_t(a.splits) * uint32_t(a.b.kv_heads);
    const auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3(grid), dim3(256), 0, s, a);
    };
    // bytes that one workgroup reads past the caches: decode_long 41.1 us -> 38.9, decode_batch 145.8 -> 136.4; not for heads of
    // 256, whose lanes take 32 bytes in two loads (56.5 us of drafted rows -> 57.9)
    if (!a.few && a.softcap > 0.0f) go(attend_many_kernel<T, D, true>);
    else if (!a.few) go(attend_many_kernel<T, D, false>);
    else if (D < 256 && a.tiles == 1) go(attend_few_kernel<T, D, (D < 256)>);
    else go(attend_few_kernel<T, D, false>);
    if (a.splits > 1) {
        const int64_t heads = int64_t(a.b.rows) * a.q_heads;
        const auto join = [&](auto kernel, int64_t groups) {
            hipLaunchKernelGGL(kernel, dim3(uint32_t(groups)), dim3(256), 0, s, a);
        };
        if (a.splits > 16) join(attend_join_kernel<T, D>, heads);
        else join(attend_join_few_kernel<T, D>, (heads * (D / 4) + 255) / 256);
    }
    return hipGetLastError();
}
template <class T>
hipError_t attend_type(const AttendArgs& a, hipStream_t s) {
    switch (a.b.dim) {
    case 64: return attend_go<T, 64>(a, s);
    case 128: return attend_go<T, 128>(a, s);
    case 256: return attend_go<T, 256>(a, s);
    default: return hipErrorInvalidValue;
    }
}

}  // namespace

hipError_t launch_attend(const AttendArgs& a, hipStream_t s) {
    switch (a.type) {
    case kActF16: return attend_type<f16>(a, s);
    case kActBF16: return attend_type<bf16>(a, s);
    default: return hipErrorInvalidValue;
    }
}

}  // namespace dev
}  // namespace xl
