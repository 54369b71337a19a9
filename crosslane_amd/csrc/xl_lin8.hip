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
// Channels are the result's rows, tokens its columns: a lane has neighbouring
// channels of one token.
//
// Two kernels: lin8_rows_kernel for few tokens, bound by the weights' bytes and
// latency, and lin8_tile_kernel, bound by the matrix cores, or by the bytes that
// come from L2 to LDS where tiles are small. What they cost stands in kWays.
#include <hip/hip_ext.h>

#include <algorithm>
#include <cmath>
#include <iterator>
#include <type_traits>
#include <utility>

#include "xl_act.hpp"
#include "xl_dev.hpp"

namespace xl::dev {
namespace {

typedef int v4i __attribute__((ext_vector_type(4)));

// The clamps are comparisons that a NaN fails, so it stays one: fminf and fmaxf return the
// other operand, and a row with a NaN scale would come out as finite numbers.
__device__ __forceinline__ float swiglu1(float g, float u, float lim) {
    if (lim > 0.0f) {
        g = g > lim ? lim : g;
        u = u > lim ? lim : u < -lim ? -lim : u;
    }
    return __fdiv_rn(g, 1.0f + expf(-g)) * u;
}

// Eight XCDs take workgroups in turn. Tile of workgroup b so that each XCD works on a
// run of consecutive tiles, ordered in groups eight token tiles deep: the 32 workgroups
// that an XCD's CUs run at a time are 8 x 4 tiles, and its L2 serves four of five reads.
__device__ __forceinline__ void tile_of(int b, int tm, int tn, int& m, int& n) {
    const int all = tm * tn, x = b & 7, per = all >> 3, rest = all & 7;
    b = x * per + min(x, rest) + (b >> 3);
    constexpr int GM = 8;
    const int in_group = GM * tn, g = b / in_group, first = g * GM, deep = min(tm - first, GM);
    const int r = b - g * in_group;
    m = first + r % deep;
    n = r / deep;
}

template <int I>
using index = std::integral_constant<int, I>;
template <int N, class F>
__device__ __forceinline__ void each(F&& f) {   // f(0), ... f(N - 1) with compile-time arguments
    [&]<int... I>(std::integer_sequence<int, I...>) { (f(index<I>{}), ...); }(std::make_integer_sequence<int, N>{});
}

// `n` rows of K bytes from row `first`, as a buffer whose range ends with the last
// row's last 16 bytes (nothing behind it is read).
__device__ __forceinline__ v4i rows_of(const int8_t* p, int64_t stride, int64_t first, int64_t n, int K) {
    const uint64_t at = reinterpret_cast<uint64_t>(p + first * stride);
    const uint32_t bytes = uint32_t((n - 1) * stride) + uint32_t((K + 15) & ~15);
    return v4i{__builtin_amdgcn_readfirstlane(int(uint32_t(at))), __builtin_amdgcn_readfirstlane(int(uint32_t(at >> 32) & 0xffffu)),
               __builtin_amdgcn_readfirstlane(int(bytes)), 0x00020000};
}
// Its 16 bytes at voff + soff straight to LDS, lane by lane from `lds` on. Neither a
// register's value nor, for the compiler, an access to LDS: left to it, every read of
// LDS behind such a load waits for all of them. wait_loads and the barriers here order
// loads and reads instead; with the "memory" that each names nothing moves across them.
// (m0 is nobody else's here, and a register that a statement cannot name. The scalar
// operands come from the scalar unit; a vector instruction's would need five wait states,
// which the compiler does not put before a statement: tests/test_lin8_code.py looks for them.)
__device__ __forceinline__ void buffer16_lds(v4i r, const int8_t* lds, uint32_t voff, int soff) {
    const uint32_t at = uint32_t(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) const int8_t*)lds));
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
                 :: "s"(__builtin_amdgcn_readfirstlane(int(at))), "v"(voff), "s"(r), "s"(soff) : "memory");
}
// All but the last N of the wave's loads to LDS are there.
template <int N>
__device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(%0)" :: "n"(N) : "memory"); }
// The wave's reads of LDS are done; then the workgroup's barrier.
__device__ __forceinline__ void reads_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// A mask of 16 bytes, the first n kept.
__device__ __forceinline__ v4i bytes_below(int n) {
    v4i m;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int left = n - 4 * i;
        m[i] = left >= 4 ? -1 : left <= 0 ? 0 : (1 << (8 * left)) - 1;
    }
    return m;
}

// TT tokens x TC channels (of each matrix) per workgroup, WT x WC waves, S stages of
// 128 bytes of K in LDS, OCC waves to a SIMD. Row m of a wave's tile i is channel
// 4 NI (m / 4) + 4 i + m % 4 of the wave's, so that a lane has 4 NI consecutive channels
// and a token's are stored in runs of 16 NI.
//
// Loads go straight to LDS: 55 bytes a clock and CU arrive this way where 32 go through
// registers and ds_write, and rows are loaded in whole 128-byte lines (64-byte pieces: 27).
// LDS gives 240 a clock to the waves' reads, no bank conflicts. 8192 x 8192 x 8192 takes
// 406 us (2.71 POP/s of 5; random values, which pull the clock below 2 GHz; all zeros
// 303 us), 8192 x 5120 x (2 x 4096) with SwiGLU 287 us, by registers 334.
template <class OT, bool GATED, int TT, int TC, int WT, int WC, int S, int R, int OCC>
__global__ __launch_bounds__(64 * WT * WC, OCC) void lin8_tile_kernel(Lin8Args a, int tm, int tn) {
    constexpr int BK = 128, NT = 64 * WT * WC, M = GATED ? 2 : 1;
    constexpr int WTT = TT / WT, WTC = TC / WC;            // a wave's tokens and channels
    constexpr int NJ = WTT / 16, NI = WTC / 16;
    constexpr int RPL = NT / 8;                            // rows of one load of all threads
    constexpr int LT = (TT + RPL - 1) / RPL, LC = (TC + RPL - 1) / RPL;   // 16-byte loads of a thread
    constexpr bool SPARE = TT % RPL || TC % RPL;           // the last ones of some waves bring nothing
    constexpr int PARTS = S == 2 ? 2 : 1;                  // parts of a stage's tokens that are given back by themselves
    static_assert(R <= NJ && NJ % R == 0 && S >= 2 && S <= 4 && LT % PARTS == 0 && NJ % PARTS == 0);
    constexpr int STAGE = (TT + M * TC) * BK;
    __shared__ alignas(16) int8_t lds0[STAGE], lds1[STAGE], lds2[S > 2 ? STAGE : 16], lds3[S > 3 ? STAGE : 16], spare[SPARE ? 1024 : 16];
    const auto stage = [&](auto si) -> int8_t* {
        constexpr int i = decltype(si)::value % S;
        if constexpr (i == 0) return lds0;
        else if constexpr (i == 1) return lds1;
        else if constexpr (i == 2) return lds2;
        else return lds3;
    };
    const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c = lane & 15, q = lane >> 4;
    const int wt = wv / WC, wc = wv % WC;
    int bm, bn;
    tile_of(blockIdx.x, tm, tn, bm, bn);
    const int64_t t0 = int64_t(bm) * TT, n0 = int64_t(bn) * TC;
    // rows behind the last one are out of the buffers' range
    const auto xr = rows_of(a.x, a.x_stride, t0, min(int64_t(TT), a.T - t0), a.K);
    const auto wr = rows_of(a.w, a.w_stride, n0, min(int64_t(TC), a.N - n0), a.K);
    const auto ur = rows_of(GATED ? a.up : a.w, a.w_stride, n0, min(int64_t(TC), a.N - n0), a.K);
    // A load brings 8 rows of 128 bytes, lane by lane one behind the other in LDS; chunk p
    // of row r lies at p ^ (r & 7), so that 16 rows of one chunk meet no bank twice.
    const int row = tid >> 3, k16 = 16 * ((tid ^ row) & 7);
    uint32_t offt[LT], offc[LC];
#pragma unroll
    for (int i = 0; i < LT; ++i) {
        const int r = row + i * RPL, in = r % (TT / PARTS);   // PARTS 2: the waves' first tiles in the first half of the rows
        offt[i] = uint32_t(in / (WTT / PARTS) * WTT + r / (TT / PARTS) * (WTT / PARTS) + in % (WTT / PARTS)) * uint32_t(a.x_stride) + k16;
    }
#pragma unroll
    for (int i = 0; i < LC; ++i) {
        const int r = row + i * RPL, in = r % WTC, m = in & 15;   // LDS row r: tile in / 16 of wave r / WTC, row m
        offc[i] = uint32_t(r / WTC * WTC + 4 * NI * (m >> 2) + 4 * (in >> 4) + (m & 3)) * uint32_t(a.w_stride) + k16;
    }
    const int steps = (a.K + BK - 1) / BK;
    constexpr int L = LT + M * LC;
    // Load i of stage `si`; behind the rows' end nothing is read, but the count stays.
    const auto load = [&](auto si, auto ii, int s) {
        constexpr int i = decltype(ii)::value, j = i < LT ? i : (i - LT) % LC, rows = i < LT ? TT : TC;
        constexpr int part = i < LT ? 0 : i < LT + LC ? TT : TT + TC;
        int8_t* b = stage(si) + (part + j * RPL + wv * 8) * BK;
        const int k = min(s * BK, a.K);   // never behind the buffer's range
        uint32_t out = s * BK + k16 < a.K ? 0u : 0x80000000u;
        if constexpr ((j + 1) * RPL > rows)
            if (j * RPL + wv * 8 >= rows) {
                b = spare;
                out = 0x80000000u;
            }
        if constexpr (i < LT) buffer16_lds(xr, b, offt[j] | out, k);
        else if constexpr (i < LT + LC) buffer16_lds(wr, b, offc[j] | out, k);
        else buffer16_lds(ur, b, offc[j] | out, k);
    };
    v4i acc[M][NI][NJ] = {};
    v4i fw[2][M][NI], ft[R];
    const uint32_t gett = uint32_t((wt * (WTT / PARTS) + c) * BK), getc = uint32_t((TT + wc * WTC + c) * BK);
    const uint32_t at[2] = {uint32_t(16 * (q ^ (c & 7))), uint32_t(16 * ((4 + q) ^ (c & 7)))};
    const auto weights = [&](auto hi, const int8_t* b) {   // of the step's half h
        constexpr int h = decltype(hi)::value;
#pragma unroll
        for (int m = 0; m < M; ++m)
#pragma unroll
            for (int i = 0; i < NI; ++i) fw[h][m][i] = *reinterpret_cast<const v4i*>(b + getc + (m * TC + 16 * i) * BK + at[h]);
    };
    const auto tokens = [&](auto pi, const int8_t* b) {    // piece p: half p / NJ, token tile p % NJ
        constexpr int p = decltype(pi)::value;
        constexpr int j = p % NJ, JP = NJ / PARTS;
        ft[p % R] = *reinterpret_cast<const v4i*>(b + gett + (j / JP * (TT / PARTS) + 16 * (j % JP)) * BK + at[p / NJ]);
    };
    const auto multiply = [&](auto pi) {
        constexpr int p = decltype(pi)::value, h = p / NJ, j = p % NJ;
#pragma unroll
        for (int m = 0; m < M; ++m)
#pragma unroll
            for (int i = 0; i < NI; ++i)
                acc[m][i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fw[h][m][i], ft[p % R], acc[m][i][j], 0, 0, 0);
    };
    // A step reads its 2 NJ pieces R ahead of their products; the last R products run
    // after the barrier, over the next step's first reads. The loads lie between the
    // products, as a wave that issues them in a row stands still until the memory pipeline
    // has taken them.
    //
    // S > 2: a step loads the stage S - 1 ahead, into the one that every wave has read when
    // the barrier before lets it pass. S == 2: each part of a stage is given back by a
    // barrier of its own as soon as it has been read, and loaded for two steps on: the
    // weights after the first products, the first half of the tokens where the second
    // half's last reads are left, the second half at the next step's start. So every load
    // has a whole step to arrive.
    constexpr int WEIGHTS = M * LC, AHEAD = S == 2 ? WEIGHTS + LT / 2 : (S - 2) * L;   // loads on their way at a step's end
    constexpr int GIVE_T = NJ + NJ / 2 - R, GIVE_W = std::min(2, GIVE_T);               // pieces before which parts are given back
    const auto some = [&](auto si, auto fi, auto ti, int s) {   // loads from .. to - 1
        constexpr int from = decltype(fi)::value, n = std::max(0, decltype(ti)::value - from);
        each<n>([&](auto i) { load(si, index<from + i>{}, s); });
    };
    const auto piece = [&](auto si, auto xi, int s) {   // x of 2 NJ: what is loaded behind it
        constexpr int x = decltype(xi)::value;
        if constexpr (S > 2) {   // in the step's first half
            some(index<si + S - 1>{}, index<std::min(L, x * L / NJ)>{}, index<std::min(L, (x + 1) * L / NJ)>{}, s + S - 1);
        } else if constexpr (x < R) {
            some(index<si + 1>{}, index<LT / 2 + x * (LT / 2) / R>{}, index<LT / 2 + (x + 1) * (LT / 2) / R>{}, s + 1);
        } else {
            constexpr int p = x - R, w = p - GIVE_W, t = p - GIVE_T;
            constexpr int over = std::min(4, 2 * NJ - R - GIVE_W), per = (WEIGHTS + over - 1) / over;   // pieces that they lie behind
            if constexpr (w >= 0 && w < over) some(si, index<LT + std::min(WEIGHTS, w * per)>{}, index<LT + std::min(WEIGHTS, (w + 1) * per)>{}, s + 2);
            if constexpr (t >= 0 && t < 2) some(si, index<t * (LT / 2) / 2>{}, index<(t + 1) * (LT / 2) / 2>{}, s + 2);
        }
        __builtin_amdgcn_sched_barrier(0);   // the compiler would move each read to its use
    };
    const auto step = [&](auto si, int s) {
        int8_t* b = stage(si);
        if (s == steps - 1 && (a.K & (BK - 1))) {   // what lies behind a token's row counts as zeros
            const v4i keep = bytes_below(a.K - s * BK - k16);
#pragma unroll
            for (int i = 0; i < LT; ++i)
                if (TT % RPL == 0 || row + i * RPL < TT) *reinterpret_cast<v4i*>(b + tid * 16 + i * RPL * BK) &= keep;
            lds_barrier();
        }
        weights(index<0>{}, b);
        each<R>([&](auto r) {
            if (s > 0) multiply(index<2 * NJ - R + r>{});
            tokens(index<r>{}, b);
            piece(si, r, s);
        });
        each<2 * NJ - R>([&](auto p) {
            if constexpr (p == (S == 2 ? 0 : NJ - R)) weights(index<1>{}, b);
            multiply(p);
            if constexpr (S == 2 && (p == GIVE_W || p == GIVE_T)) reads_barrier();
            tokens(index<p + R>{}, b);
            piece(si, index<p + R>{}, s);
        });
        // this wave's part of the next stage is here, and its reads of this one are done
        wait_loads<AHEAD>();
        reads_barrier();
    };
    if constexpr (S == 2) {
        some(index<0>{}, index<0>{}, index<L>{}, 0);
        some(index<1>{}, index<LT>{}, index<L>{}, 1);
        some(index<1>{}, index<0>{}, index<LT / 2>{}, 1);
    } else {
        each<S - 1>([&](auto si) { some(si, index<0>{}, index<L>{}, si); });
    }
    wait_loads<AHEAD>();
    reads_barrier();
    for (int s = 0; s < steps; s += S) each<S>([&](auto si) { if (s + si < steps) step(si, s + si); });
    each<R>([&](auto r) { multiply(index<2 * NJ - R + r>{}); });
    wait_loads<0>();   // none writes LDS behind the workgroup's end
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
        const auto put = [&](auto ei, auto ni) {   // channels e0 .. e0 + N - 1
            constexpr int e0 = decltype(ei)::value, N = decltype(ni)::value;
            float y[N];
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const int i = (e0 + e) / 4;
                y[e] = float(acc[0][i][j][e & 3]) * xs * ws[0][e0 + e];
                if constexpr (GATED) y[e] = swiglu1(y[e], float(acc[1][i][j][e & 3]) * xs * ws[1][e0 + e], a.lim);
            }
            if (left > e0) store_rounded<OT, N>(o + e0, left - e0, y);
        };
        each<NI / 2>([&](auto i) { put(index<8 * i>{}, index<8>{}); });
        if constexpr (NI % 2) put(index<4 * NI - 4>{}, index<4>{});
    }
}

// Four results of a token to an output of any type.
__device__ __forceinline__ void store4(const Lin8Args& a, int64_t t, int64_t n, int left, const float (&y)[4]) {
    const auto put = [&](auto* o) {
        using OT = std::remove_pointer_t<decltype(o)>;
        o += t * a.out_stride + n;
        OT v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = rounded<OT>(y[e]);
        if (left >= 4) {
            __builtin_memcpy(o, v, sizeof v);
        } else {
#pragma unroll
            for (int e = 0; e < 3; ++e)
                if (e < left) o[e] = v[e];
        }
    };
    if (a.out_type == kActF32) put(static_cast<float*>(a.out));
    else if (a.out_type == kActF16) put(static_cast<f16*>(a.out));
    else put(static_cast<bf16*>(a.out));
}

// Few tokens: 16 NJ of them and 16 NI channels (of each matrix) per workgroup. The
// waves take the rows' 128-byte pieces in turn, each through a ring of U stages of its
// own in LDS (no barrier; loads of whole 128-byte lines go straight there, as in the
// tile kernel), and their sums are added in LDS at the end.
// XT: type of x; other than int8, the one row of x is quantized into LDS by every
// workgroup, while its first weights are on their way (4096 x 5120: 7.2 us, 9.8 with a
// launch of its own; two rows gain nothing). The quants lie on 16 bytes: behind the odd
// end of the small arrays, every read of them was split (7.9 us; 1024 x 16384 13.9 for 9.7).
//
// Bound by the weights' bytes, latency and launch: 4096 x 5120 in 6.1 us for one to 8.1
// for 64 tokens (21 MB, 4.4 us at the rate of a copy). With the operands straight from
// memory to registers, 16 rows of 64 bytes an instruction, it was 6.2 and 12.3.
template <int NI, int NJ, bool GATED, int XT, int NW, int U>
__global__ __launch_bounds__(64 * NW) void lin8_rows_kernel(Lin8Args a) {
    constexpr int M = GATED ? 2 : 1, NT = 64 * NW, BK = 128;
    constexpr bool FUSED = XT != kActI8;
    static_assert(!FUSED || NJ == 1);
    static_assert(U >= 2 && U <= 4);
    constexpr int XR = FUSED ? 0 : 16 * NJ;                     // rows of x in a stage, ahead of the weights'
    constexpr int STAGE = (XR + M * NI * 16) * BK, L = STAGE / 1024;
    __shared__ alignas(16) int8_t lds0[NW][STAGE], lds1[NW][STAGE], lds2[U > 2 ? NW : 1][U > 2 ? STAGE : 16], lds3[U > 3 ? NW : 1][U > 3 ? STAGE : 16];
    static_assert(sizeof(lds0) >= size_t(NW) * M * NI * NJ * 1024, "the sums take the first stage's place");
    alignas(16) extern __shared__ int8_t xq[];                  // FUSED: K rounded up to 128; read 16 bytes at a time
    __shared__ float red[16], scale1;
    const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c = lane & 15, q = lane >> 4;
    const auto stage = [&](auto ui) -> int8_t* {
        constexpr int u = decltype(ui)::value;
        if constexpr (u == 0) return lds0[wv];
        else if constexpr (u == 1) return lds1[wv];
        else if constexpr (u == 2) return lds2[wv];
        else return lds3[wv];
    };
    const int64_t t0 = int64_t(blockIdx.y) * (16 * NJ), n0 = int64_t(blockIdx.x) * (16 * NI);
    const auto xr = rows_of(FUSED ? a.w : a.x, FUSED ? 16 : a.x_stride, FUSED ? 0 : t0, FUSED ? 1 : min(int64_t(16 * NJ), a.T - t0), FUSED ? 16 : a.K);
    const auto wr = rows_of(a.w, a.w_stride, n0, min(int64_t(16 * NI), a.N - n0), a.K);
    const auto ur = rows_of(GATED ? a.up : a.w, a.w_stride, n0, min(int64_t(16 * NI), a.N - n0), a.K);
    // a load: 8 rows, chunk p of row r at p ^ (r & 7)
    const int row = lane >> 3, k16 = 16 * ((lane ^ row) & 7);
    const uint32_t offx = uint32_t(row) * uint32_t(a.x_stride) + k16, offw = uint32_t(row) * uint32_t(a.w_stride) + k16;
    const auto load = [&](auto ui, int p) {   // behind the rows' end nothing is read, but the count stays
        int8_t* b = stage(ui);
        const int k = min(p * BK, a.K);
        const uint32_t out = p * BK + k16 < a.K ? 0u : 0x80000000u;
        if constexpr (!FUSED)
#pragma unroll
            for (int j = 0; j < 2 * NJ; ++j) buffer16_lds(xr, b + j * 1024, (offx + 8 * j * uint32_t(a.x_stride)) | out, k);
#pragma unroll
        for (int i = 0; i < 2 * NI; ++i) buffer16_lds(wr, b + XR * BK + i * 1024, (offw + 8 * i * uint32_t(a.w_stride)) | out, k);
        if constexpr (GATED)
#pragma unroll
            for (int i = 0; i < 2 * NI; ++i) buffer16_lds(ur, b + (XR + 16 * NI) * BK + i * 1024, (offw + 8 * i * uint32_t(a.w_stride)) | out, k);
    };
    using XF = std::conditional_t<XT == kActF32, float, std::conditional_t<XT == kActF16, f16, bf16>>;
    const XF* x = reinterpret_cast<const XF*>(a.x);
    constexpr int FIRST = FUSED ? 2 : 1;
    float first[FIRST][8];
    if constexpr (FUSED)   // ahead of the weights, as loads are waited for in their order
#pragma unroll
        for (int i = 0; i < FIRST; ++i) load8(x + 8 * (tid + i * NT), a.K - 8 * (tid + i * NT), first[i]);
    each<U>([&](auto u) { load(u, wv + u * NW); });
    if constexpr (FUSED) {
        float v[8], m = 0.0f;
#pragma unroll
        for (int i = 0; i < FIRST; ++i) m = amax8(first[i], m);
        for (int at = 8 * (tid + FIRST * NT); at < a.K; at += 8 * NT) {
            load8(x + at, a.K - at, v);
            m = amax8(v, m);
        }
        const float d = row_scale(group_join<true>(m, red), a.err);
        if (tid == 0) scale1 = d;
        const int end = (a.K + BK - 1) / BK * BK;
#pragma unroll
        for (int i = 0; i < FIRST; ++i)
            if (8 * (tid + i * NT) < end) store_quants(xq + 8 * (tid + i * NT), first[i], d);
        for (int at = 8 * (tid + FIRST * NT); at < end; at += 8 * NT) {
            load8(x + at, a.K - at, v);
            store_quants(xq + at, v, d);
        }
        lds_barrier();
    }
    v4i acc[M][NI][NJ] = {};
    const int pieces = (a.K + BK - 1) / BK;
    const uint32_t at[2] = {uint32_t(c * BK + 16 * (q ^ (c & 7))), uint32_t(c * BK + 16 * ((4 + q) ^ (c & 7)))};
    const auto work = [&](auto ui, int p) {
        const int8_t* b = stage(ui);
        v4i fw[2][M][NI], fx[2][NJ];
        wait_loads<(U - 1) * L>();
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int j = 0; j < NJ; ++j)
                fx[h][j] = FUSED ? *reinterpret_cast<const v4i*>(xq + p * BK + 64 * h + 16 * q) : *reinterpret_cast<const v4i*>(b + 16 * j * BK + at[h]);
#pragma unroll
            for (int m = 0; m < M; ++m)
#pragma unroll
                for (int i = 0; i < NI; ++i) fw[h][m][i] = *reinterpret_cast<const v4i*>(b + (XR + 16 * (m * NI + i)) * BK + at[h]);
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // read: the stage is free
        load(ui, p + U * NW);
        if (!FUSED && p == pieces - 1 && (a.K & (BK - 1))) {   // what lies behind a token's row counts as zeros
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const v4i keep = bytes_below(a.K - p * BK - 64 * h - 16 * q);
#pragma unroll
                for (int j = 0; j < NJ; ++j) fx[h][j] &= keep;
            }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int j = 0; j < NJ; ++j)
#pragma unroll
                for (int m = 0; m < M; ++m)
#pragma unroll
                    for (int i = 0; i < NI; ++i)
                        acc[m][i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fw[h][m][i], fx[h][j], acc[m][i][j], 0, 0, 0);
    };
    for (int p = wv; p < pieces; p += U * NW) each<U>([&](auto u) { if (p + u * NW < pieces) work(u, p + u * NW); });
    wait_loads<0>();   // none is left to write into a stage
    __syncthreads();
    v4i* sums = reinterpret_cast<v4i*>(&lds0[0][0]);   // [wave][tile][lane]
    constexpr int TILES = M * NI * NJ;
#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
            for (int j = 0; j < NJ; ++j) sums[(wv * TILES + (m * NI + i) * NJ + j) * 64 + lane] = acc[m][i][j];
    __syncthreads();
    // item: tile i, j and lane of its results
    for (int it = tid; it < NI * NJ * 64; it += NT) {
        const int tile = it >> 6, i = tile / NJ, j = tile % NJ;
        const int64_t t = t0 + 16 * j + c, n = n0 + 16 * i + 4 * q;
        if (t >= a.T || n >= a.N) continue;
        v4i s[M];
#pragma unroll
        for (int m = 0; m < M; ++m) {
            s[m] = sums[(m * NI * NJ + tile) * 64 + lane];
#pragma unroll
            for (int w = 1; w < NW; ++w) s[m] += sums[(w * TILES + m * NI * NJ + tile) * 64 + lane];
        }
        const int left = int(min(int64_t(4), int64_t(a.N) - n));
        float xs;
        if constexpr (FUSED) xs = scale1;
        else xs = a.x_scale[t];
        float y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int64_t r = n + min(e, left - 1);
            y[e] = float(s[0][e]) * xs * a.w_scale[r];
            if constexpr (GATED) y[e] = swiglu1(y[e], float(s[M - 1][e]) * xs * a.up_scale[r], a.lim);
        }
        store4(a, t, n, left, y);
    }
}

template <class OT, bool GATED, int TT, int TC, int WT, int WC, int S, int R, int OCC>
void lin8_tiles(const Lin8Args& a, hipStream_t s, hipEvent_t stop) {
    const int tm = (a.T + TT - 1) / TT, tn = (a.N + TC - 1) / TC;
    hipExtLaunchKernelGGL((lin8_tile_kernel<OT, GATED, TT, TC, WT, WC, S, R, OCC>), dim3(tm * tn), dim3(64 * WT * WC), 0, s, nullptr, stop, 0, a, tm, tn);
}

template <int NI, int NJ, bool GATED, int XT, int NW, int U>
void lin8_rows(const Lin8Args& a, hipStream_t s, hipEvent_t stop) {
    const size_t lds = XT == kActI8 ? 0 : size_t((a.K + 127) & ~127);
    hipExtLaunchKernelGGL((lin8_rows_kernel<NI, NJ, GATED, XT, NW, U>), dim3((a.N + 16 * NI - 1) / (16 * NI), (a.T + 16 * NJ - 1) / (16 * NJ)),
                          dim3(64 * NW), lds, s, nullptr, stop, 0, a);
}
// The ways to run a call, in order of their tiles: tokens, channels (of each of one or
// two matrices), workgroups that one CU holds, and the microseconds that they take:
// fixed, and for each 128-byte step of K with the chip mostly idle and with a workgroup
// on every CU. Fitted to calls of 1 to 8192 tokens, 64 to 8192 k, 100 to 9216 channels,
// one and two matrices. Over 284 of them, each run all ways (in graphs, 16 calls), the way
// of the least estimate is 0.9 % slower than the fastest on average. Where it errs most:
// 8192 x (2 x 100) with 1,024 to 2,048 tokens, 14 to 38 % (25.8 for 18.8 us); 5120 x (2 x
// 4096) with 48 and 64 tokens, 19 and 20 % (13.6 for 11.4); 5120 x 4096 with 17 to 32, 17 to
// 19 % (7.4 for 6.3). The next one is 9 %.
struct Way {
    int tokens, one, two, per_cu;   // two 0: one matrix only
    float fixed, idle, busy;
    bool rows;   // lin8_rows_kernel, whose workgroups overlap; else lin8_tile_kernel, in rounds over the CUs
};
constexpr Way kWays[] = {
    {16, 16, 16, 1, 3.4f, 0.047f, 0.078f, true},    {32, 16, 16, 1, 3.4f, 0.077f, 0.110f, true},
    {32, 32, 0, 1, 3.6f, 0.086f, 0.152f, true},     {32, 64, 32, 1, 4.6f, 0.135f, 0.213f, true},
    {64, 64, 32, 2, 3.3f, 0.250f, 0.609f, false},   {64, 128, 64, 1, 3.3f, 0.309f, 0.323f, false},
    {128, 128, 64, 1, 4.9f, 0.442f, 0.551f, false}, {128, 160, 96, 1, 6.0f, 0.576f, 0.742f, false},
    {128, 256, 128, 1, 7.8f, 0.685f, 1.005f, false}, {256, 160, 0, 1, 9.1f, 0.752f, 1.258f, false},
    {256, 192, 96, 1, 9.1f, 1.145f, 1.415f, false}, {256, 256, 128, 1, 11.6f, 1.124f, 1.871f, false},
};
constexpr float kRowsRound = 0.8f, kTilesRound = 4.2f;   // ... for each further round
int lin8_way(const Lin8Args& a, int cus) {
    if (a.x_type != kActI8) return 0;
    int best = 0;
    float least = 0.0f;
    for (int i = 0; i < int(std::size(kWays)); ++i) {
        const Way& w = kWays[i];
        const int64_t ch = a.up ? w.two : w.one;
        if (ch == 0) continue;
        const float per = float(((a.T + w.tokens - 1) / w.tokens) * ((a.N + ch - 1) / ch)) / float(cus * w.per_cu);
        const float rounds = w.rows ? std::max(per, 1.0f) : std::ceil(per);
        const float us = w.fixed + (w.rows ? kRowsRound : kTilesRound) * (rounds - 1.0f) +
                         float((a.K + 127) / 128) * std::max((w.rows ? 1.0f : rounds) * w.idle, per * w.busy);
        if (i == 0 || us < least) {
            best = i;
            least = us;
        }
    }
    return best;
}

template <class OT, bool GATED>
void lin8_tiled(const Lin8Args& a, int way, hipStream_t s, hipEvent_t stop) {
    constexpr int G = GATED ? 2 : 1;
    switch (way) {
    case 4: return lin8_tiles<OT, GATED, 64, 64 / G, 4, 1, 4, 1, 2>(a, s, stop);
    case 5: return lin8_tiles<OT, GATED, 64, 128 / G, 2, 4, 4, 2, 2>(a, s, stop);
    case 6: return lin8_tiles<OT, GATED, 128, 128 / G, 4, 2, 4, 2, 2>(a, s, stop);
    case 7: return lin8_tiles<OT, GATED, 128, GATED ? 96 : 160, 4, 2, GATED ? 3 : 4, 2, 2>(a, s, stop);
    case 8: return lin8_tiles<OT, GATED, 128, 256 / G, 2, 4, 3, 4, 2>(a, s, stop);
    case 9:
        if constexpr (!GATED) return lin8_tiles<OT, GATED, 256, 160, 4, 2, 3, 4, 2>(a, s, stop);
        break;
    case 10: return lin8_tiles<OT, GATED, 256, 192 / G, 4, 2, 2, 4, 2>(a, s, stop);
    default: break;
    }
    lin8_tiles<OT, GATED, 256, 256 / G, 2, 4, 2, 4, 2>(a, s, stop);
}
template <bool GATED>
void lin8_run(const Lin8Args& a, int way, hipStream_t s, hipEvent_t stop) {
    if (a.x_type == kActF32) return lin8_rows<1, 1, GATED, kActF32, 8, 2>(a, s, stop);
    if (a.x_type == kActF16) return lin8_rows<1, 1, GATED, kActF16, 8, 2>(a, s, stop);
    if (a.x_type == kActBF16) return lin8_rows<1, 1, GATED, kActBF16, 8, 2>(a, s, stop);
    switch (way) {
    case 0: return lin8_rows<1, 1, GATED, kActI8, 8, 2>(a, s, stop);
    case 1: return lin8_rows<1, 2, GATED, kActI8, 4, GATED ? 2 : 3>(a, s, stop);
    case 2:
        if constexpr (!GATED) return lin8_rows<2, 2, GATED, kActI8, 8, 2>(a, s, stop);
        break;
    case 3: return lin8_rows<GATED ? 2 : 4, 2, GATED, kActI8, 4, 3>(a, s, stop);
    default: break;
    }
    if (a.out_type == kActF32) lin8_tiled<float, GATED>(a, way, s, stop);
    else if (a.out_type == kActF16) lin8_tiled<f16, GATED>(a, way, s, stop);
    else lin8_tiled<bf16, GATED>(a, way, s, stop);
}

}  // namespace

hipError_t launch_lin8(const Lin8Args& a, int cus, hipStream_t s, hipEvent_t stop) {
    if (a.T < 1 || a.T > kLinMaxT || a.N < 1 || a.K < 1 || a.K > kLinMaxK || a.w_stride % 16 ||
        (a.x_type == kActI8 ? a.x_stride % 16 != 0 : !lin8_quantizes(a.T, a.K)))
        return hipErrorInvalidValue;
    if (a.out_type < kActF32 || a.out_type > kActBF16) return hipErrorInvalidValue;
    const int way = lin8_way(a, cus);
    if (a.up) lin8_run<true>(a, way, s, stop);
    else lin8_run<false>(a, way, s, stop);
    return hipGetLastError();
}

}  // namespace xl::dev
