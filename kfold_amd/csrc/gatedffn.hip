// Gated feed-forward block, forward and backward, for training.
// Reference: src/kfold/model/layers/folding/transition.py:48-68 without its layer norm,
// primitives/activation.py:20-29 (SwiGLU).
//
//   [u; v] = x W_in^T (W_in [2F, C]),   h = silu(u) * v,   y = h W_out^T (W_out [C, F])
//   dh = dy W_out;  s = sigmoid(u);  dv = dh u s;  du = dh v s (1 + u (1 - s))
//   dx = [du dv] W_in;  dW_in = [du dv]^T x;  dW_out = dy^T h
//
// Nothing but x is kept for the backward pass: u, v are computed again (4 of its 16 M C F
// operations), which costs less than writing and reading them.
//
// Arithmetic.  bf16 tensors: products on the matrix cores with fp32 accumulation; h, du and dv are
// rounded to bf16 because they are operands of the next product (half a step, 2^-8 of the value at most,
// on terms of a sum; the results are rounded to bf16 anyway); everything else stays fp32.  fp32 tensors:
// every operand is split into three bf16 parts (split3, once per call) and the six part products with
// i + j <= 2 are summed, which carries fp32 accuracy; h, du, dv are kept as three parts as well.
#include "ffn_tiles.hpp"

namespace kfh {

// fp32 values -> their three split3 planes, `n` bf16 apart: 8 values per thread, up to four tensors
struct SplitArgs { const float* src[4]; uint16_t* dst[4]; long long n[4]; };
__global__ __launch_bounds__(256) void ffn_split_kernel(SplitArgs p) {
    const int t = blockIdx.y;
    const long long n = p.n[t];
    for (long long i = ((long long)blockIdx.x * 256 + threadIdx.x) * 8; i < n; i += (long long)gridDim.x * 2048) {
        float x[8], q[8][3];
        load8<KFH_F32>(p.src[t], (size_t)i, x);
#pragma unroll
        for (int e = 0; e < 8; ++e) split3(x[e], q[e]);
#pragma unroll
        for (int k = 0; k < 3; ++k)
            *reinterpret_cast<u32x4*>(p.dst[t] + k * n + i) = u32x4{pack_bf16(q[0][k], q[1][k]), pack_bf16(q[2][k], q[3][k]),
                                                                   pack_bf16(q[4][k], q[5][k]), pack_bf16(q[6][k], q[7][k])};
    }
}

// ---------------------------------------------------------------------------------------------
// Hidden values of a tile of TM rows x 64 hidden channels; wavefront (wm, wn) owns TM / 2 rows x 32
// channels of u and v (and dh: the same accumulator shape, from dy and w_out).
//   forward : h [M, F]
//   backward: d [M, 2F] = (du, dv) and h [M, F]
// Operands and results in P parts, consecutive planes.  The next D k-tiles travel from memory while the
// matrix cores work on the present one.
// ---------------------------------------------------------------------------------------------
template <int P, int TM> constexpr int hidden_lds() {
    constexpr int BK = P == 3 ? 32 : 64;
    const int in = P * (TM + 128) * (BK + 8) * 2;
    const int out = P * TileStore<KFH_BF16, TM, 64, 256>::BYTES;
    return in > out ? in : out;
}

template <int P, bool BWD, int TM>
__global__ __launch_bounds__(256) void ffn_hidden_kernel(const uint16_t* __restrict__ x, const uint16_t* __restrict__ dy,
                                                         const uint16_t* __restrict__ w_in,
                                                         const uint16_t* __restrict__ w_out, uint16_t* __restrict__ h,
                                                         uint16_t* __restrict__ d, long long M, int C, int F) {
    constexpr int BK = P == 3 ? 32 : 64, LDK = BK + 8, NA = TM / 64, D = P == 1 && TM == 64 ? 2 : 1;
    __shared__ __attribute__((aligned(16))) char smem[hidden_lds<P, TM>()];
    uint16_t* const sa = reinterpret_cast<uint16_t*>(smem);
    uint16_t* const su = sa + P * TM * LDK;
    uint16_t* const sv = su + P * 64 * LDK;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int wm = wave & 1, wn = wave >> 1;
    long long mt;
    int ft;
    if (!xcd_tile(blockIdx.x, (M + TM - 1) / TM, (F + 63) / 64, mt, ft)) return;
    const long long m0 = mt * TM;
    const int f0 = ft * 64;
    f32x16 u[NA][1], v[NA][1], g[NA][1];
    zero_acc(u); zero_acc(v); zero_acc(g);
    using X = TileLoad<K_MAJOR, TM, BK, P, 256>;
    using W = TileLoad<K_MAJOR, 64, BK, P, 256>;
    using WT = TileLoad<R_MAJOR, 64, BK, P, 256>;
    X lx, ly;
    W lu, lv;
    WT lo;
    lx.init(x, C, M * C * 2, m0, M, tid);
    lu.init(w_in, C, 4LL * F * C, f0, F, tid);
    lv.init(w_in, C, 4LL * F * C, (long long)F + f0, 2LL * F, tid);
    if constexpr (BWD) {
        ly.init(dy, C, M * C * 2, m0, M, tid);
        lo.init(w_out, F, 2LL * F * C, f0, F, tid);
    }
    typename X::Regs rx[D];
    typename W::Regs ru[D], rv[D];
    typename WT::Regs ro[D];
    const int n = (C + BK - 1) / BK;                        // steps [0, n): x, u and v; [n, 2n): dy, dh
    auto fetch = [&](int s, auto set) {
        constexpr int I = decltype(set)::v;
        if (s < n) {
            lx.fetch((long long)s * BK, C, tid, rx[I]);
            lu.fetch((long long)s * BK, C, tid, ru[I]);
            lv.fetch((long long)s * BK, C, tid, rv[I]);
        } else if (BWD && s < 2 * n) {
            ly.fetch((long long)(s - n) * BK, C, tid, rx[I]);
            lo.fetch((long long)(s - n) * BK, C, tid, ro[I]);
        }
    };
    auto first = [&](int s, auto set) {
        constexpr int I = decltype(set)::v;
        __syncthreads();
        X::commit(sa, tid, rx[I]); W::commit(su, tid, ru[I]); W::commit(sv, tid, rv[I]);
        __syncthreads();
        fetch(s + D, set);
        tile_mma<P, NA, 1, TM, 64, BK>(sa, wm * (TM / 2), su, wn * 32, lane, u);
        tile_mma<P, NA, 1, TM, 64, BK>(sa, wm * (TM / 2), sv, wn * 32, lane, v);
    };
    auto second = [&](int s, auto set) {
        constexpr int I = decltype(set)::v;
        __syncthreads();
        X::commit(sa, tid, rx[I]); WT::commit(su, tid, ro[I]);
        __syncthreads();
        fetch(s + D, set);
        tile_mma<P, NA, 1, TM, 64, BK>(sa, wm * (TM / 2), su, wn * 32, lane, g);
    };
    fetch(0, Int<0>{});
    if constexpr (D == 1) {
        for (int s = 0; s < n; ++s) first(s, Int<0>{});
        if constexpr (BWD)
            for (int s = n; s < 2 * n; ++s) second(s, Int<0>{});
    } else {
        fetch(1, Int<1>{});
        // register set = parity of the step; with an odd n the dy steps begin with set 1
        for (int s = 0; s < n; s += 2) {
            first(s, Int<0>{});
            if (s + 1 < n) first(s + 1, Int<1>{});
        }
        if constexpr (BWD) {
            if (n & 1) second(n, Int<1>{});
            for (int s = n + (n & 1); s < 2 * n; s += 2) {
                second(s, Int<0>{});
                if (s + 1 < 2 * n) second(s + 1, Int<1>{});
            }
        }
    }
    // h, du and dv in the places of dh, u and v (forward: h in the place of u)
#pragma unroll
    for (int a = 0; a < NA; ++a)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const float uu = u[a][0][e], vv = v[a][0][e];
            const float s = sigmoidf_fast(uu), us = uu * s;
            if constexpr (BWD) {
                const float gg = g[a][0][e];
                g[a][0][e] = us * vv;
                u[a][0][e] = gg * vv * (s + us * (1.f - s));
                v[a][0][e] = gg * us;
            } else {
                u[a][0][e] = us * vv;
            }
        }
    using Out = TileStore<KFH_BF16, TM, 64, 256>;
    auto write = [&](const f32x16(&t)[NA][1], uint16_t* dst, long long ld) {      // planes M * ld apart
        __syncthreads();
#pragma unroll
        for (int a = 0; a < NA; ++a) {
            const int r = wm * (TM / 2) + 32 * a + (lane & 31);
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int f = wn * 32 + 8 * q + 4 * (lane >> 5);
                float s[4][3];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    s[e][0] = t[a][0][4 * q + e];
                    if constexpr (P == 3) split3(t[a][0][4 * q + e], s[e]);
                }
#pragma unroll
                for (int k = 0; k < P; ++k) Out::put(smem + k * Out::BYTES, r, f, s[0][k], s[1][k], s[2][k], s[3][k]);
            }
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < P; ++k) Out::flush(smem + k * Out::BYTES, dst + (size_t)k * M * ld, ld, m0, M, f0, F, tid);
    };
    if constexpr (BWD) {
        write(g, h, F);
        write(u, d, 2LL * F);
        write(v, d + F, 2LL * F);
    } else {
        write(u, h, F);
    }
}

// ---------------------------------------------------------------------------------------------
// out[m][n] = sum_k A(m, k) B(n, k), operands in P parts (planes `ap`, `bp` bytes apart); AK / BK_ as
// TileLoad's KIND; a workgroup of NW wavefronts owns TM x TN results, wavefront (wm, wn) TM / WM x TN / WN
// of them.  The contraction is cut into `splits` ranges of kper; with OUT_PART the results are fp32 partial
// tiles at out + range * (Mo + Mo2) * No, and Mo2 more rows may come from a second pair of operands of the same
// kinds (both weight gradients in one launch).
//
// What bounds it with many rows is the way of the operands into LDS: with 128 x 128 tiles the weight
// gradient 2048 x 256 over 146689 rows takes 261 us for the loads alone, 100 us for the products alone
// (1.5 PF/s) and 272 us together; a 256 x 256 tile asks for half the bytes: 213 us.
// ---------------------------------------------------------------------------------------------
template <int TM, int TN> struct Waves {                     // wavefronts of a tile and their arrangement
    static constexpr int NW = TM * TN >= 256 * 128 ? 8 : 4;
    static constexpr int WM = NW == 4 || TM <= TN ? 2 : 4, WN = NW / WM;
};
// results: fp32 partial tiles of a range of the contraction, or the product itself in bf16 or fp32
enum : int { OUT_BF16 = KFH_BF16, OUT_F32 = KFH_F32, OUT_PART };
template <int P, int TM, int TN, int OUT> struct GemmLds {
    static constexpr int BK = P == 3 ? 32 : 64, NT = Waves<TM, TN>::NW * 64;
    using Out = TileStore<OUT == OUT_BF16 ? (int)KFH_BF16 : (int)KFH_F32, TM, TN / Waves<TM, TN>::WN, NT>;  // one column of wavefronts
    static constexpr int IN = 2 * P * (TM + TN) * (BK + 8) * 2;
    static constexpr int BYTES = IN > Out::BYTES ? IN : Out::BYTES;
};

template <int P, int AK, int BK_, int OUT, int TM, int TN>
__device__ __forceinline__ void gemm_tile(
    const void* __restrict__ A, long long lda, long long ap, const void* __restrict__ B, long long ldb, long long bp,
    void* __restrict__ out, long long Mo, int No, long long K, long long kper, int splits, const void* __restrict__ A2,
    long long lda2, long long ap2, const void* __restrict__ B2, int Mo2) {
    using W = Waves<TM, TN>;
    using Lds = GemmLds<P, TM, TN, OUT>;
    constexpr bool PART = OUT == OUT_PART;
    constexpr int BK = Lds::BK, LDK = BK + 8, NT = Lds::NT;
    constexpr int RM = TM / W::WM, RN = TN / W::WN, NA = RM / 32, NB = RN / 32;
    // k-tiles on their way in registers: the small tiles are used where there are few workgroups and the
    // latency of the loads is what counts; the large ones have no registers for more than one
    constexpr int D = TM == 64 ? (P == 3 ? 2 : 4) : 1;
    __shared__ __attribute__((aligned(16))) char smem[Lds::BYTES];
    constexpr int BUF = P * (TM + TN) * LDK;
    uint16_t* const buf = reinterpret_cast<uint16_t*>(smem);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int wm = wave % W::WM, wn = wave / W::WM;
    const long long mtiles1 = (Mo + TM - 1) / TM, mtiles = mtiles1 + (PART ? (Mo2 + TM - 1) / TM : 0);
    const int ntiles = (No + TN - 1) / TN;
    // tiles that share operand rows follow each other on one XCD: those of a row tile, or (PART) all
    // tiles of one range of the contraction
    long long mt, z = 0;
    int nt;
    if constexpr (PART) {
        int t;
        if (!xcd_tile(blockIdx.x, splits, (int)(mtiles * ntiles), z, t)) return;
        mt = t / ntiles;
        nt = t % ntiles;
    } else {
        if (!xcd_tile(blockIdx.x, mtiles, ntiles, mt, nt)) return;
    }
    char* base = static_cast<char*>(out) + (PART ? (size_t)z * (Mo + Mo2) * No * 4 : 0);
    if (PART && mt >= mtiles1) {
        mt -= mtiles1;
        base += (size_t)Mo * No * 4;
        A = A2; lda = lda2; ap = ap2; B = B2; Mo = Mo2;
    }
    const long long m0 = mt * TM;
    const int n0 = nt * TN;
    const long long kb = z * kper, ke = min(kb + kper, K);
    f32x16 acc[NA][NB];
    zero_acc(acc);
    using LA = TileLoad<AK, TM, BK, P, NT>;
    using LB = TileLoad<BK_, TN, BK, P, NT>;
    LA la;
    LB lb;
    typename LA::Regs ra[D];
    typename LB::Regs rb[D];
    la.init(A, lda, ap, m0, Mo, tid);
    lb.init(B, ldb, bp, n0, No, tid);
    // while the matrix cores work on a k-tile in LDS, the next is written to the other LDS buffer and D more
    // travel from memory to registers; one barrier per k-tile
    const long long steps = kb < ke ? (ke - kb + BK - 1) / BK : 0;
    auto fetch = [&](long long s, auto set) {
        constexpr int I = decltype(set)::v % D;
        if (s >= steps) return;
        la.fetch(kb + s * BK, ke, tid, ra[I]);
        lb.fetch(kb + s * BK, ke, tid, rb[I]);
    };
    auto commit = [&](long long s, auto set) {
        constexpr int I = decltype(set)::v % D;
        if (s >= steps) return;
        uint16_t* const b = buf + (s & 1) * BUF;
        LA::commit(b, tid, ra[I]);
        LB::commit(b + P * TM * LDK, tid, rb[I]);
    };
    auto step = [&](long long s, auto next) {                 // next: register set of step s + 1
        commit(s + 1, next);
        fetch(s + 1 + D, next);
        const uint16_t* const b = buf + (s & 1) * BUF;
        tile_mma<P, NA, NB, TM, TN, BK>(b, wm * RM, b + P * TM * LDK, wn * RN, lane, acc);
        __syncthreads();
    };
    fetch(0, Int<0>{});
    if constexpr (D > 1) fetch(1, Int<1>{});
    if constexpr (D > 2) { fetch(2, Int<2>{}); fetch(3, Int<3>{}); }
    commit(0, Int<0>{});
    fetch(D, Int<0>{});
    __syncthreads();
    for (long long s = 0; s < steps; s += D) {
        step(s, Int<1>{});
        if constexpr (D > 1)
            if (s + 1 < steps) step(s + 1, Int<2>{});
        if constexpr (D > 2) {
            if (s + 2 < steps) step(s + 2, Int<3>{});
            if (s + 3 < steps) step(s + 3, Int<4>{});
        }
    }
    // through LDS, one column of wavefronts at a time
    using Out = typename Lds::Out;
#pragma unroll 1
    for (int c = 0; c < W::WN; ++c) {
        if (c) __syncthreads();
        if (wn == c) {
#pragma unroll
            for (int a = 0; a < NA; ++a)
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        Out::put(smem, wm * RM + 32 * a + (lane & 31), 32 * b + 8 * q + 4 * (lane >> 5), acc[a][b][4 * q],
                                 acc[a][b][4 * q + 1], acc[a][b][4 * q + 2], acc[a][b][4 * q + 3]);
        }
        __syncthreads();
        Out::flush(smem, base, No, m0, Mo, n0 + c * RN, No, tid);
    }
}
// a name per workgroup size
template <int P, int AK, int BK_, int OUT, int TM, int TN>
__global__ __launch_bounds__(256) void ffn_gemm_kernel(
    const void* __restrict__ A, long long lda, long long ap, const void* __restrict__ B, long long ldb, long long bp,
    void* __restrict__ out, long long Mo, int No, long long K, long long kper, int splits, const void* __restrict__ A2,
    long long lda2, long long ap2, const void* __restrict__ B2, int Mo2) {
    gemm_tile<P, AK, BK_, OUT, TM, TN>(A, lda, ap, B, ldb, bp, out, Mo, No, K, kper, splits, A2, lda2, ap2, B2, Mo2);
}
template <int P, int AK, int BK_, int OUT, int TM, int TN>
__global__ __launch_bounds__(512) void ffn_gemm_large_kernel(
    const void* __restrict__ A, long long lda, long long ap, const void* __restrict__ B, long long ldb, long long bp,
    void* __restrict__ out, long long Mo, int No, long long K, long long kper, int splits, const void* __restrict__ A2,
    long long lda2, long long ap2, const void* __restrict__ B2, int Mo2) {
    gemm_tile<P, AK, BK_, OUT, TM, TN>(A, lda, ap, B, ldb, bp, out, Mo, No, K, kper, splits, A2, lda2, ap2, B2, Mo2);
}

// ---------------------------------------------------------------------------------------------
// The two products of a forward call in bf16 with few rows, where nothing but latency counts: a workgroup
// owns 32 x 32 results, its wavefronts take the k-steps in turn and read their fragments straight from memory
// (every load of a batch independent of the others), and the partial sums meet in LDS.
//   GATED: out[m][n] = silu(A W_n) * (A W_{N+n});  else out[m][n] = A W_n;   A [M, K], W [N or 2N, K]
// ---------------------------------------------------------------------------------------------
constexpr int kSmallWaves = 4, kSmallBatch = 4;

template <bool GATED>
__global__ __launch_bounds__(64 * kSmallWaves) void ffn_small_kernel(const uint16_t* __restrict__ A,
                                                                     const uint16_t* __restrict__ W,
                                                                     uint16_t* __restrict__ out, long long M, int N, int K) {
    constexpr int NB = GATED ? 2 : 1;
    __shared__ float red[kSmallWaves][NB][16][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 31, half = lane >> 5;
    const long long m0 = (long long)blockIdx.y * 32;
    const int n0 = blockIdx.x * 32;
    const uint16_t* const a = A + (size_t)min(m0 + col, M - 1) * K;
    const uint16_t* const b = W + (size_t)min(n0 + col, N - 1) * K;
    f32x16 acc[NB];
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
        for (int v = 0; v < 16; ++v) acc[j][v] = 0.f;
    const int steps = (K + 15) / 16;
    for (int s = wave; s < steps; s += kSmallWaves * kSmallBatch) {
        u32x4 fa[kSmallBatch], fb[kSmallBatch][NB];
#pragma unroll
        for (int i = 0; i < kSmallBatch; ++i) {
            const int k = min((s + i * kSmallWaves) * 16 + 8 * half, K - 8);
            fa[i] = *reinterpret_cast<const u32x4*>(a + k);
#pragma unroll
            for (int j = 0; j < NB; ++j) fb[i][j] = *reinterpret_cast<const u32x4*>(b + (size_t)j * N * K + k);
        }
#pragma unroll
        for (int i = 0; i < kSmallBatch; ++i) {
            // a k-step (or its upper half) behind the end: A's values count as zeros
            const bool in = (s + i * kSmallWaves) * 16 + 8 * half < K;
            const bf16x8 x = __builtin_bit_cast(bf16x8, in ? fa[i] : u32x4{0u, 0u, 0u, 0u});
#pragma unroll
            for (int j = 0; j < NB; ++j)
                acc[j] = mfma32(__builtin_bit_cast(bf16x8, in ? fb[i][j] : u32x4{0u, 0u, 0u, 0u}), x, acc[j]);
        }
    }
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
        for (int v = 0; v < 16; ++v) red[wave][j][v][lane] = acc[j][v];
    __syncthreads();
    // wavefront q finishes accumulator rows 4q .. 4q + 3: four consecutive columns of one row per lane
    float o[NB][4];
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            o[j][e] = 0.f;
#pragma unroll
            for (int w = 0; w < kSmallWaves; ++w) o[j][e] += red[w][j][4 * wave + e][lane];
        }
    if constexpr (GATED) {
#pragma unroll
        for (int e = 0; e < 4; ++e) o[0][e] = o[0][e] * sigmoidf_fast(o[0][e]) * o[1][e];
    }
    const int n = n0 + 8 * wave + 4 * half;
    if (m0 + col < M && n < N) store4<KFH_BF16>(out, (size_t)(m0 + col) * N + n, o[0][0], o[0][1], o[0][2], o[0][3]);
}

// Sums of `parts` partial matrices [R1 + R2, C]: the first R1 rows go to out1 as they are, the other R2 rows
// transposed to out2 [C, R2]; either may be null.  32 x 32 values per workgroup, its four groups of 256 threads take
// every fourth part; a fixed order.  A launch takes two such sums of the same C, of rows of tiles [0, tiles) and
// those behind (the weight gradients' and dx's of a backward call with few rows: 82.6 against 84.8 us at
// 666 x 384 x 768 in fp32, 31.9 against 33.8 at 37 x 384 x 768 in bf16).
struct SumArgs { const float* part; int parts; long long R1; int R2, C; void* out1; void* out2; };
template <int IO>
__device__ __forceinline__ void sum_tile(const SumArgs& p, long long tile, float (&red)[4][32][36]) {
    const int t = threadIdx.x & 255, grp = threadIdx.x >> 8;
    const long long tiles1 = (p.R1 + 31) / 32;
    const bool second = tile >= tiles1;
    const long long r0 = (second ? tile - tiles1 : tile) * 32, rows = second ? p.R2 : p.R1;
    const int c0 = blockIdx.x * 32, rr = t >> 3, cc = (t & 7) * 4;
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
    if (r0 + rr < rows && c0 + cc < p.C) {
        const size_t n = (size_t)(p.R1 + p.R2) * p.C, at = (size_t)((second ? p.R1 : 0) + r0 + rr) * p.C + c0 + cc;
#pragma unroll 4
        for (int z = grp; z < p.parts; z += 4) {
            const f32x4 w = *reinterpret_cast<const f32x4*>(p.part + z * n + at);
#pragma unroll
            for (int e = 0; e < 4; ++e) s[e] += w[e];
        }
    }
    *reinterpret_cast<f32x4*>(&red[grp][rr][cc]) = s;
    __syncthreads();
    if (grp != 0) return;
    float o[4];
    if (!second) {
        if (!p.out1 || r0 + rr >= rows || c0 + cc >= p.C) return;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = (red[0][rr][cc + e] + red[1][rr][cc + e]) + (red[2][rr][cc + e] + red[3][rr][cc + e]);
        store4<IO>(p.out1, (size_t)(r0 + rr) * p.C + c0 + cc, o[0], o[1], o[2], o[3]);
    } else {
        // column rr of the tile, its rows cc .. cc + 3
        if (!p.out2 || r0 + cc >= rows || c0 + rr >= p.C) return;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = (red[0][cc + e][rr] + red[1][cc + e][rr]) + (red[2][cc + e][rr] + red[3][cc + e][rr]);
        store4<IO>(p.out2, (size_t)(c0 + rr) * p.R2 + r0 + cc, o[0], o[1], o[2], o[3]);
    }
}
template <int IO, int IO2>
__global__ __launch_bounds__(1024) void ffn_sum_parts_kernel(SumArgs p, unsigned tiles, SumArgs q) {
    __shared__ float red[4][32][36];
    if (blockIdx.y < tiles) sum_tile<IO>(p, blockIdx.y, red);
    else sum_tile<IO2>(q, blockIdx.y - tiles, red);
}

// ---------------------------------------------------------------------------------------------
static size_t up256(size_t x) { return (x + 255) / 256 * 256; }
static long long up_div(long long a, long long b) { return (a + b - 1) / b; }

// Tile of a product [a, b]: the larger, the fewer bytes per result come into LDS; 256 along a side that has
// 256, 128 else, as long as every CU gets a workgroup (`more`: ranges the contraction may be cut into), or
// 64 x 64.  fp32 stays with 64 x 64: its operands take three times the LDS.
struct Tile { int m, n; };
static Tile pick_tile(long long a, long long b, long long more, int io_dtype) {
    if (io_dtype != KFH_BF16) return {64, 64};
    auto full = [&](int m, int n) { return up_div(a, m) * up_div(b, n) * more >= 256; };
    const int m = a >= 256 ? 256 : 128, n = b >= 256 ? 256 : 128;
    if (full(m, n)) return {m, n};
    if (full(128, 128)) return {128, 128};
    return {64, 64};
}

// Both weight gradients are one product [2F + F, C] over the rows: (du, dv)^T x and h^T dy.  Ranges of rows that are
// summed in parallel: one workgroup per CU with large tiles (as many as fit; more would only add partial sums),
// two with the others, at least 256 rows each.
struct Wgrad { Tile t; int splits; long long per; };
static Wgrad wgrad_plan(long long M, long long a1, long long a2, long long b, int io_dtype) {
    Wgrad w;
    const long long most = max(1LL, up_div(M, 256));
    w.t = pick_tile(a1 + a2, b, most, io_dtype);
    const long long tiles = (up_div(a1, w.t.m) + up_div(a2, w.t.m)) * up_div(b, w.t.n);
    w.splits = (int)min(min(max(1LL, (w.t.m * w.t.n > 128 * 128 ? 256 : 512) / tiles), most), 256LL);
    // whole rounds over the XCDs, unless more than a tenth of the workgroups went (2048 + 1024 channels of d and h
    // by 256, 21 ranges: 313 us counted through, 362 with 16 ranges dealt to the XCDs; 146689 rows)
    if (const int r = w.splits / 8 * 8; r * 10 >= w.splits * 9) w.splits = r;
    w.per = up_div(up_div(M, w.splits), 64) * 64;
    return w;
}
static size_t wgrad_part_bytes(long long M, int C, int F, int io_dtype) {
    return (size_t)wgrad_plan(M, 2LL * F, F, C, io_dtype).splits * 3 * F * C * 4;
}

// A product with few tiles and a long contraction is cut into ranges of it (at least 8 k-tiles each, from
// 24 on, towards two workgroups per CU): 666 x 384 with K = 1536 in fp32 took 90 us in one piece.
static int product_splits(long long Mo, long long No, long long K, int io_dtype) {
    const long long BK = io_dtype == KFH_F32 ? 32 : 64, steps = up_div(K, BK);
    if (steps < 24) return 1;
    const long long tiles = up_div(Mo, 64) * up_div(No, 64);
    return (int)max(1LL, min(512 / tiles, steps / 8));
}
static size_t product_part_bytes(long long Mo, long long No, long long K, int io_dtype) {
    const int s = product_splits(Mo, No, K, io_dtype);
    return s > 1 ? (size_t)s * Mo * No * 4 : 0;
}

// The streamed kernels: bf16, a width they are built for, whole steps of hidden channels, and 16384 rows, which
// give them 128 workgroups of 128 rows (C <= 128) or 64 of 256 rows (C = 256): fewer leave too many of the 256 CUs
// idle.  Tiles against streamed kernels, us, forward | backward:
//     C x F          8192 rows                 16384                     32768                     65536
//     64 x 128       12.3 12.2 | 25.5 24.8     12.2 12.0 | 34.5 29.1     12.1 11.7 | 38.9 35.3     19.1 11.9 | 53.5 46.8
//     128 x 256      12.3 14.3 | 40.1 40.4     14.8 14.7 | 44.0 43.8     18.6 15.5 | 60.7 53.1     34.8 20.4 | 92.1 76.8
//     128 x 512      15.3 22.9 | 45.7 56.1     21.2 23.2 | 64.5 63.6     31.1 24.4 | 94.1 81.3     56.6 31.9 | 160 124
//     256 x 512      19.2 44.8 | 59.9 95.7     26.2 44.6 | 88.3 110      44.7 52.5 | 137 135       80.7 71.2 | 274 201
//     256 x 1024     28.5 76.0 | 96.9 162      46.1 77.0 | 144 179       79.7 86.9 | 269 228       148 123 | 520 365
// so the two meet at the threshold for C = 64 and 128, and at 256 only between 32768 and 49152 rows: there the calls
// from 16384 rows up to that pay up to 1.7 times the tiles' time.
static bool streamed(long long M, int C, int F, int io_dtype) {
    return io_dtype == KFH_BF16 && (C == 64 || C == 128 || C == 256) && F % 32 == 0 && M >= 16384;
}

// Few rows: with fewer than 128 tiles of 64 x 64 hidden values the kernels that work straight from memory are
// faster (37 x 384 x 768: 10.8 against 14.8 us; 666 rows, 132 tiles: equal; 1000 rows: 20.4 against 13.6).
static bool few_rows(long long M, int F) { return up_div(M, 64) * up_div(F, 64) < 128; }

// Workspace: h [M, F] (not in a fused forward call), backward: d [M, 2F], row-major in P planes or (streamed)
// in blocks; packed weights of the streamed kernels; planes of x, w_in, w_out and dy (fp32); partial sums of y or dx
// and of the weight gradients
struct FfnWs { size_t h, d, pack, x, wi, wo, dy, part, wpart, total; };
static FfnWs ffn_ws(long long M, int C, int F, int backward, int io_dtype) {
    const size_t e = io_dtype == KFH_F32 ? 6 : 2, split = io_dtype == KFH_F32 ? 6 : 0;
    const bool st = streamed(M, C, F, io_dtype), fused = st && C <= 128;
    const size_t rows = st ? (size_t)up_div(M, 32) * 32 : (size_t)M;         // whole blocks
    FfnWs w;
    size_t at = 0;
    auto take = [&](size_t bytes) { const size_t a = at; at += up256(bytes); return a; };
    w.h = take(backward || !fused ? rows * F * e : 0);
    w.d = take(backward ? rows * 2 * F * e : 0);
    w.pack = take(st ? ffn_stream_pack_bytes(C, F, backward) : 0);
    w.x = take((size_t)M * C * split);
    w.wi = take((size_t)2 * F * C * split);
    w.wo = take((size_t)F * C * split);
    w.dy = take(backward ? (size_t)M * C * split : 0);
    w.part = take(st ? 0 : product_part_bytes(M, C, backward ? 2LL * F : F, io_dtype));
    w.wpart = take(backward ? wgrad_part_bytes(M, C, F, io_dtype) : 0);
    w.total = at;
    return w;
}
size_t gated_ffn_ws_bytes(long long M, int C, int F, int backward, int io_dtype) {
    return ffn_ws(M, C, F, backward, io_dtype).total;
}

// p's results in p_dtype, q's in IO; either may have no parts
template <int IO>
static void sum_parts(SumArgs p, int p_dtype, const SumArgs& q, hipStream_t stream) {
    auto tiles = [](const SumArgs& a) { return a.parts ? (unsigned)(up_div(a.R1, 32) + up_div(a.R2, 32)) : 0u; };
    if (!p.parts && !q.parts) return;
    const dim3 grid((unsigned)up_div(p.parts ? p.C : q.C, 32), tiles(p) + tiles(q));
    if (p_dtype == KFH_BF16) hipLaunchKernelGGL((ffn_sum_parts_kernel<KFH_BF16, IO>), grid, dim3(1024), 0, stream, p, tiles(p), q);
    else hipLaunchKernelGGL((ffn_sum_parts_kernel<KFH_F32, IO>), grid, dim3(1024), 0, stream, p, tiles(p), q);
}

template <int P, bool BWD>
static void hidden(const void* x, const void* dy, const void* w_in, const void* w_out, void* h, void* d, long long M, int C,
                   int F, hipStream_t stream) {
    const int nt = (int)up_div(F, 64);
    auto run = [&](auto tm) {
        constexpr int TM = decltype(tm)::v;
        hipLaunchKernelGGL((ffn_hidden_kernel<P, BWD, TM>), dim3(xcd_grid(up_div(M, TM), nt)), dim3(256), 0, stream,
                           static_cast<const uint16_t*>(x), static_cast<const uint16_t*>(dy), static_cast<const uint16_t*>(w_in),
                           static_cast<const uint16_t*>(w_out), static_cast<uint16_t*>(h), static_cast<uint16_t*>(d), M, C, F);
    };
    if constexpr (P == 1) {
        if (up_div(M, 128) * nt >= 256) return run(Int<128>{});
    }
    run(Int<64>{});
}

// an operand: its first part, elements per row, bytes between parts
struct Operand { const void* p; long long ld, plane; };

template <int P, int AK, int BK_, int OUT, int TM, int TN>
static void gemm(Operand a, Operand b, void* out, long long Mo, int No, long long K, long long kper, int splits,
                 hipStream_t stream, Operand a2 = {}, Operand b2 = {}, int Mo2 = 0) {
    const long long mt = up_div(Mo, TM) + up_div(Mo2, TM), nt = up_div(No, TN);
    const dim3 grid(OUT == OUT_PART ? xcd_grid(splits, (int)(mt * nt)) : xcd_grid(mt, (int)nt));
    if constexpr (Waves<TM, TN>::NW == 8)
        hipLaunchKernelGGL((ffn_gemm_large_kernel<P, AK, BK_, OUT, TM, TN>), grid, dim3(512), 0, stream, a.p, a.ld, a.plane, b.p, b.ld,
                           b.plane, out, Mo, No, K, kper, splits, a2.p, a2.ld, a2.plane, b2.p, Mo2);
    else
        hipLaunchKernelGGL((ffn_gemm_kernel<P, AK, BK_, OUT, TM, TN>), grid, dim3(256), 0, stream, a.p, a.ld, a.plane, b.p, b.ld, b.plane,
                           out, Mo, No, K, kper, splits, a2.p, a2.ld, a2.plane, b2.p, Mo2);
}

// out [Mo, No] = A [Mo, K] (AK) times B, [No, K] (K_MAJOR) or [K, No] (R_MAJOR); part: product_part_bytes.
// Returns the sum that is left to do, if the contraction was cut.
template <int P, int AK, int BK_>
static SumArgs product(Operand a, Operand b, void* out, float* part, long long Mo, int No, long long K, hipStream_t stream) {
    constexpr int IO = P == 3 ? KFH_F32 : KFH_BF16;
    const Tile t = pick_tile(Mo, No, 1, IO);
    if constexpr (AK == K_BLOCK) {                          // streamed calls: 16384 rows of 256 channels at least
        // (y: 128 rows a tile, 256 leave the compiler three registers short)
        constexpr int TM = BK_ == K_MAJOR ? 128 : 256;
        if (t.m == 256) gemm<P, AK, BK_, IO, TM, 256>(a, b, out, Mo, No, K, K, 1, stream);
        else gemm<P, AK, BK_, IO, 128, 128>(a, b, out, Mo, No, K, K, 1, stream);
        return {};
    } else {
        const int splits = product_splits(Mo, No, K, IO);
        if (splits > 1) {
            const long long BK = P == 3 ? 32 : 64, per = up_div(up_div(K, BK), splits) * BK;
            gemm<P, AK, BK_, OUT_PART, 64, 64>(a, b, part, Mo, No, K, per, splits, stream);
            return {part, splits, Mo, 0, No, out, nullptr};
        }
        bool done = false;
        if constexpr (P == 1) {
            done = true;
            if (t.n == 256) gemm<P, AK, BK_, IO, 256, 256>(a, b, out, Mo, No, K, K, 1, stream);
            else if (t.m == 256) gemm<P, AK, BK_, IO, 256, 128>(a, b, out, Mo, No, K, K, 1, stream);
            else if (t.m == 128) gemm<P, AK, BK_, IO, 128, 128>(a, b, out, Mo, No, K, K, 1, stream);
            else done = false;
        }
        if (!done) gemm<P, AK, BK_, IO, 64, 64>(a, b, out, Mo, No, K, K, 1, stream);
        return {};
    }
}

// dw_in [2F, C] = d^T x and dw_out [C, F] = (h^T dy)^T; d and h of kind AK (R_MAJOR or R_BLOCK); either result may
// be null, its rows are then left out.  Returns the sum of the partial products, which is left to do.
template <int P, int AK>
static SumArgs wgrad(Operand d, Operand x, Operand h, Operand dy, float* part, void* dw_in, void* dw_out, long long M, int C,
                     int F, hipStream_t stream) {
    if (!dw_in && !dw_out) return {};
    const int Ma = dw_in ? 2 * F : F, Mb = dw_in && dw_out ? F : 0;
    const Wgrad w = wgrad_plan(M, 2LL * F, F, C, P == 3 ? KFH_F32 : KFH_BF16);
    auto run = [&](auto tm, auto tn) {
        gemm<P, AK, R_MAJOR, OUT_PART, decltype(tm)::v, decltype(tn)::v>(dw_in ? d : h, dw_in ? x : dy, part, Ma, C, M, w.per, w.splits,
                                                                        stream, h, dy, Mb);
    };
    bool done = false;
    if constexpr (P == 1) {
        done = true;
        if (w.t.m == 256 && w.t.n == 256) run(Int<256>{}, Int<256>{});
        else if (w.t.m == 256) run(Int<256>{}, Int<128>{});
        else if (w.t.n == 256) run(Int<128>{}, Int<256>{});
        else if (w.t.m == 128) run(Int<128>{}, Int<128>{});
        else done = false;
    }
    if (!done) run(Int<64>{}, Int<64>{});
    // (dw_out alone: no direct rows)
    return {part, w.splits, dw_in ? 2LL * F : 0, dw_out ? F : 0, C, dw_in, dw_out};
}

// the three planes of the fp32 operands
static void split_operands(const void* x, const void* w_in, const void* w_out, const void* dy, char* ws, const FfnWs& w,
                           long long M, int C, int F, hipStream_t stream) {
    SplitArgs s;
    const void* const src[4] = {x, w_in, w_out, dy};
    const size_t dst[4] = {w.x, w.wi, w.wo, w.dy};
    const long long n[4] = {M * C, 2LL * F * C, (long long)F * C, M * C};
    long long most = 0;
    for (int i = 0; i < 4; ++i) {
        s.src[i] = static_cast<const float*>(src[i]);
        s.dst[i] = reinterpret_cast<uint16_t*>(ws + dst[i]);
        s.n[i] = n[i];
        most = max(most, n[i]);
    }
    hipLaunchKernelGGL(ffn_split_kernel, dim3((unsigned)min(up_div(most, 2048), 4096LL), dy ? 4 : 3), dim3(256), 0, stream, s);
}

template <int P>
static void forward_t(const void* x, const void* w_in, const void* w_out, void* y, char* ws, long long M, int C, int F,
                      hipStream_t stream) {
    constexpr int IO = P == 3 ? KFH_F32 : KFH_BF16;
    const FfnWs w = ffn_ws(M, C, F, 0, IO);
    float* const part = reinterpret_cast<float*>(ws + w.part);
    if constexpr (P == 3) {
        split_operands(x, w_in, w_out, nullptr, ws, w, M, C, F, stream);
        x = ws + w.x;
        w_in = ws + w.wi;
        w_out = ws + w.wo;
    } else if (streamed(M, C, F, KFH_BF16)) {
        launch_ffn_stream(x, nullptr, w_in, w_out, ws + w.pack, ws + w.h, nullptr, y, M, C, F, stream);
        if (C > 128) product<1, K_BLOCK, K_MAJOR>({ws + w.h, F, 0}, {w_out, F, 0}, y, part, M, C, F, stream);
        return;
    }
    if constexpr (P == 1) {
        if (few_rows(M, F)) {
            const uint16_t* const xs = static_cast<const uint16_t*>(x);
            uint16_t* const h = reinterpret_cast<uint16_t*>(ws + w.h);
            hipLaunchKernelGGL(ffn_small_kernel<true>, dim3((unsigned)up_div(F, 32), (unsigned)up_div(M, 32)), dim3(64 * kSmallWaves), 0,
                               stream, xs, static_cast<const uint16_t*>(w_in), h, M, F, C);
            hipLaunchKernelGGL(ffn_small_kernel<false>, dim3((unsigned)up_div(C, 32), (unsigned)up_div(M, 32)), dim3(64 * kSmallWaves), 0,
                               stream, h, static_cast<const uint16_t*>(w_out), static_cast<uint16_t*>(y), M, C, F);
            return;
        }
    }
    hidden<P, false>(x, nullptr, w_in, nullptr, ws + w.h, nullptr, M, C, F, stream);
    const SumArgs left = product<P, K_MAJOR, K_MAJOR>({ws + w.h, F, M * F * 2}, {w_out, F, 2LL * F * C}, y, part, M, C, F, stream);
    sum_parts<IO>({}, IO, left, stream);
}

template <int P>
static void backward_t(const void* dy, const void* x, const void* w_in, const void* w_out, void* dx, void* dw_in,
                       void* dw_out, int dw_dtype, char* ws, long long M, int C, int F, hipStream_t stream) {
    constexpr int IO = P == 3 ? KFH_F32 : KFH_BF16;
    const FfnWs w = ffn_ws(M, C, F, 1, IO);
    char* const h = ws + w.h;
    char* const d = ws + w.d;
    float* const part = reinterpret_cast<float*>(ws + w.part);
    float* const wpart = reinterpret_cast<float*>(ws + w.wpart);
    if constexpr (P == 3) {
        split_operands(x, w_in, w_out, dy, ws, w, M, C, F, stream);
        x = ws + w.x;
        w_in = ws + w.wi;
        w_out = ws + w.wo;
        dy = ws + w.dy;
    } else if (streamed(M, C, F, KFH_BF16)) {
        launch_ffn_stream(x, dy, w_in, w_out, ws + w.pack, h, d, dx, M, C, F, stream);
        const SumArgs left = wgrad<1, R_BLOCK>({d, 2LL * F, 0}, {x, C, 0}, {h, F, 0}, {dy, C, 0}, wpart, dw_in, dw_out, M, C, F, stream);
        sum_parts<IO>(left, dw_dtype, {}, stream);
        if (dx && C > 128) product<1, K_BLOCK, R_MAJOR>({d, 2LL * F, 0}, {w_in, C, 0}, dx, part, M, C, 2LL * F, stream);
        return;
    }
    hidden<P, true>(x, dy, w_in, w_out, h, d, M, C, F, stream);
    const Operand X = {x, C, M * C * 2}, DY = {dy, C, M * C * 2}, H = {h, F, M * F * 2}, D = {d, 2LL * F, M * 2 * F * 2};
    const SumArgs dw_left = wgrad<P, R_MAJOR>(D, X, H, DY, wpart, dw_in, dw_out, M, C, F, stream);
    SumArgs dx_left = {};
    if (dx) dx_left = product<P, K_MAJOR, R_MAJOR>(D, {w_in, C, 4LL * F * C}, dx, part, M, C, 2LL * F, stream);
    sum_parts<IO>(dw_left, dw_dtype, dx_left, stream);
}

void launch_gated_ffn_forward(const void* x, const void* w_in, const void* w_out, void* y, char* ws, long long M,
                              int C, int F, int io_dtype, hipStream_t stream) {
    if (io_dtype == KFH_F32) forward_t<3>(x, w_in, w_out, y, ws, M, C, F, stream);
    else forward_t<1>(x, w_in, w_out, y, ws, M, C, F, stream);
}

void launch_gated_ffn_backward(const void* dy, const void* x, const void* w_in, const void* w_out, void* dx,
                               void* dw_in, void* dw_out, int dw_dtype, char* ws, long long M, int C, int F,
                               int io_dtype, hipStream_t stream) {
    if (io_dtype == KFH_F32) backward_t<3>(dy, x, w_in, w_out, dx, dw_in, dw_out, dw_dtype, ws, M, C, F, stream);
    else backward_t<1>(dy, x, w_in, w_out, dx, dw_in, dw_out, dw_dtype, ws, M, C, F, stream);
}

}  // namespace kfh
