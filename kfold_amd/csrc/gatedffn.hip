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
// rounded to bf16 because they are operands of the next product (half a step, 2^-9 of the value, on
// terms of a sum; the results are rounded to bf16 anyway); everything else stays fp32.  fp32
// tensors: every operand is split into three bf16 parts (split3) and the six part products with
// i + j <= 2 are summed, which carries fp32 accuracy; h, du, dv are kept in fp32.
#include "train.hpp"

namespace kfh {

// ---------------------------------------------------------------------------------------------
// Operand tiles.  A tile of ROWS x BK operand values (rows: output index, k: contraction) goes
// from memory to registers to LDS, where it is stored [part][row][BK + 8] bf16, so that the 8
// k-consecutive values of an MFMA fragment are one 16-byte read; the 8 values of padding keep
// consecutive rows on different banks.
//   KC = true : memory is [row][k], k contiguous: a thread moves 8 k of a row
//   KC = false: memory is [k][row], rows contiguous: a thread loads 4 k x 8 rows and writes them
//               transposed, 4 k (8 bytes) per row
// Values outside [row < rmax, k < kmax] are zeros.
// ---------------------------------------------------------------------------------------------
template <int IO> constexpr int parts_of() { return IO == KFH_F32 ? 3 : 1; }

template <int IO, bool KC, int ROWS, int BK>
struct TileLoad {
    static constexpr int PARTS = parts_of<IO>();
    static constexpr int LDK = BK + 8;                       // bf16 per stored row
    static constexpr int PLANE = ROWS * LDK;                 // bf16 per part
    static constexpr int UNITS = KC ? ROWS * BK / 8 : ROWS * BK / 32;
    static constexpr int NU = (UNITS + 255) / 256;           // units per thread
    static constexpr int NV = KC ? 1 : 4;                    // 8-value vectors per unit
    float v[NU][NV][8];

    __device__ __forceinline__ void load(const void* src, long long ld, long long row0, long long rmax,
                                         long long k0, long long kmax, int tid) {
#pragma unroll
        for (int i = 0; i < NU; ++i) {
            const int u = i * 256 + tid;
            if constexpr (KC) {
                const long long r = row0 + u / (BK / 8), k = k0 + (u % (BK / 8)) * 8;
                const bool ok = u < UNITS && r < rmax && k < kmax;
                if (ok) load8<IO>(src, (size_t)(r * ld + k), v[i][0]);
                else
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[i][0][e] = 0.f;
            } else {
                const long long r = row0 + (u / (BK / 4)) * 8, k = k0 + (u % (BK / 4)) * 4;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const bool ok = u < UNITS && r < rmax && k + j < kmax;
                    if (ok) load8<IO>(src, (size_t)((k + j) * ld + r), v[i][j]);
                    else
#pragma unroll
                        for (int e = 0; e < 8; ++e) v[i][j][e] = 0.f;
                }
            }
        }
    }
    __device__ __forceinline__ void store(uint16_t* lds, int tid) const {
#pragma unroll
        for (int i = 0; i < NU; ++i) {
            const int u = i * 256 + tid;
            if (u >= UNITS) continue;
            if constexpr (KC) {
                uint16_t* d = lds + (u / (BK / 8)) * LDK + (u % (BK / 8)) * 8;
                if constexpr (PARTS == 1) {
                    u32x4 w;
#pragma unroll
                    for (int e = 0; e < 4; ++e) w[e] = pack_bf16(v[i][0][2 * e], v[i][0][2 * e + 1]);
                    *reinterpret_cast<u32x4*>(d) = w;
                } else {
                    float q[8][3];
#pragma unroll
                    for (int e = 0; e < 8; ++e) split3(v[i][0][e], q[e]);
#pragma unroll
                    for (int p = 0; p < 3; ++p) {
                        u32x4 w;
#pragma unroll
                        for (int e = 0; e < 4; ++e) w[e] = pack_bf16(q[2 * e][p], q[2 * e + 1][p]);
                        *reinterpret_cast<u32x4*>(d + p * PLANE) = w;
                    }
                }
            } else {
                uint16_t* d = lds + (u / (BK / 4)) * 8 * LDK + (u % (BK / 4)) * 4;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    if constexpr (PARTS == 1) {
                        u32x2 w = {pack_bf16(v[i][0][e], v[i][1][e]), pack_bf16(v[i][2][e], v[i][3][e])};
                        *reinterpret_cast<u32x2*>(d + e * LDK) = w;
                    } else {
                        float q[4][3];
#pragma unroll
                        for (int j = 0; j < 4; ++j) split3(v[i][j][e], q[j]);
#pragma unroll
                        for (int p = 0; p < 3; ++p) {
                            u32x2 w = {pack_bf16(q[0][p], q[1][p]), pack_bf16(q[2][p], q[3][p])};
                            *reinterpret_cast<u32x2*>(d + p * PLANE + e * LDK) = w;
                        }
                    }
                }
            }
        }
    }
};

// acc[i][j] += rows (a0 + 32 i) of tile `ta` times rows (b0 + 32 j) of tile `tb` over BK, as
// D[row of b][column = row of a]: a lane then holds four consecutive b indices of one a row.
template <int IO, int NA, int NB, int AROWS, int BROWS, int BK>
__device__ __forceinline__ void tile_mma(const uint16_t* ta, int a0, const uint16_t* tb, int b0, int lane,
                                         f32x16 (&acc)[NA][NB]) {
    constexpr int PARTS = parts_of<IO>(), LDK = BK + 8;
    const int col = lane & 31, half = lane >> 5;
#pragma unroll
    for (int ks = 0; ks < BK / 16; ++ks) {
        bf16x8 a[NA][PARTS], b[NB][PARTS];
#pragma unroll
        for (int p = 0; p < PARTS; ++p) {
#pragma unroll
            for (int i = 0; i < NA; ++i)
                a[i][p] = *reinterpret_cast<const bf16x8*>(ta + p * AROWS * LDK + (a0 + 32 * i + col) * LDK + ks * 16 + half * 8);
#pragma unroll
            for (int j = 0; j < NB; ++j)
                b[j][p] = *reinterpret_cast<const bf16x8*>(tb + p * BROWS * LDK + (b0 + 32 * j + col) * LDK + ks * 16 + half * 8);
        }
#pragma unroll
        for (int i = 0; i < NA; ++i)
#pragma unroll
            for (int j = 0; j < NB; ++j) {
                if constexpr (PARTS == 1) {
                    acc[i][j] = mfma32(b[j][0], a[i][0], acc[i][j]);
                } else {
                    // smallest products first
                    acc[i][j] = mfma32(b[j][2], a[i][0], acc[i][j]);
                    acc[i][j] = mfma32(b[j][0], a[i][2], acc[i][j]);
                    acc[i][j] = mfma32(b[j][1], a[i][1], acc[i][j]);
                    acc[i][j] = mfma32(b[j][1], a[i][0], acc[i][j]);
                    acc[i][j] = mfma32(b[j][0], a[i][1], acc[i][j]);
                    acc[i][j] = mfma32(b[j][0], a[i][0], acc[i][j]);
                }
            }
    }
}

template <int NA, int NB>
__device__ __forceinline__ void zero_acc(f32x16 (&acc)[NA][NB]) {
#pragma unroll
    for (int i = 0; i < NA; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
            for (int v = 0; v < 16; ++v) acc[i][j][v] = 0.f;
}

// four consecutive values of a row
template <int IO>
__device__ __forceinline__ void store4(void* base, size_t e, float a, float b, float c, float d) {
    if constexpr (IO == KFH_BF16) *reinterpret_cast<u32x2*>(static_cast<uint16_t*>(base) + e) = u32x2{pack_bf16(a, b), pack_bf16(c, d)};
    else *reinterpret_cast<f32x4*>(static_cast<float*>(base) + e) = f32x4{a, b, c, d};
}

// ---------------------------------------------------------------------------------------------
// Hidden values of a tile of 64 rows x 64 hidden channels; wavefront (wm, wn) owns 32 x 32.
//   forward : h [M, F]
//   backward: d [M, 2F] = (du, dv) and h [M, F]
// ---------------------------------------------------------------------------------------------
template <int IO, bool BWD>
__global__ __launch_bounds__(256) void ffn_hidden_kernel(const void* __restrict__ x, const void* __restrict__ dy,
                                                         const void* __restrict__ w_in,
                                                         const void* __restrict__ w_out, void* __restrict__ h,
                                                         void* __restrict__ d, long long M, int C, int F) {
    constexpr int BK = IO == KFH_F32 ? 32 : 64, LDK = BK + 8, T = 64;
    constexpr int TILE = parts_of<IO>() * T * LDK;
    __shared__ __attribute__((aligned(16))) uint16_t smem[3 * TILE];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int wm = wave & 1, wn = wave >> 1;
    const long long m0 = (long long)blockIdx.x * T;
    const int f0 = blockIdx.y * T;
    f32x16 u[1][1], v[1][1], g[1][1];
    zero_acc(u); zero_acc(v); zero_acc(g);
    TileLoad<IO, true, T, BK> lx, lu, lv;
    for (int k0 = 0; k0 < C; k0 += BK) {
        lx.load(x, C, m0, M, k0, C, tid);
        lu.load(w_in, C, f0, F, k0, C, tid);
        lv.load(w_in, C, (long long)F + f0, 2LL * F, k0, C, tid);
        __syncthreads();
        lx.store(smem, tid); lu.store(smem + TILE, tid); lv.store(smem + 2 * TILE, tid);
        __syncthreads();
        tile_mma<IO, 1, 1, T, T, BK>(smem, wm * 32, smem + TILE, wn * 32, lane, u);
        tile_mma<IO, 1, 1, T, T, BK>(smem, wm * 32, smem + 2 * TILE, wn * 32, lane, v);
    }
    if constexpr (BWD) {
        TileLoad<IO, false, T, BK> lo;
        for (int k0 = 0; k0 < C; k0 += BK) {
            lx.load(dy, C, m0, M, k0, C, tid);
            lo.load(w_out, F, f0, F, k0, C, tid);
            __syncthreads();
            lx.store(smem, tid); lo.store(smem + TILE, tid);
            __syncthreads();
            tile_mma<IO, 1, 1, T, T, BK>(smem, wm * 32, smem + TILE, wn * 32, lane, g);
        }
    }
    const long long m = m0 + wm * 32 + (lane & 31);
    if (m >= M) return;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const int f = f0 + wn * 32 + 8 * q + 4 * (lane >> 5);
        if (f >= F) continue;
        float hh[4], du[4], dv[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float uu = u[0][0][4 * q + e], vv = v[0][0][4 * q + e];
            const float s = sigmoidf_fast(uu), us = uu * s;
            hh[e] = us * vv;
            if constexpr (BWD) {
                const float gg = g[0][0][4 * q + e];
                dv[e] = gg * us;
                du[e] = gg * vv * (s + us * (1.f - s));
            }
        }
        store4<IO>(h, (size_t)m * F + f, hh[0], hh[1], hh[2], hh[3]);
        if constexpr (BWD) {
            store4<IO>(d, (size_t)m * 2 * F + f, du[0], du[1], du[2], du[3]);
            store4<IO>(d, (size_t)m * 2 * F + F + f, dv[0], dv[1], dv[2], dv[3]);
        }
    }
}

// ---------------------------------------------------------------------------------------------
// out[m][n] = sum_k A(m, k) B(n, k); AKC / BKC as TileLoad's KC.  blockIdx.z takes the contraction
// range [z * kper, (z + 1) * kper); with SPLIT the result is an fp32 partial tile at
// out + z * Mo * No, else it is written as IO.
// ---------------------------------------------------------------------------------------------
template <int IO, bool AKC, bool BKC, bool SPLIT>
__global__ __launch_bounds__(256) void ffn_gemm_kernel(const void* __restrict__ A, long long lda,
                                                       const void* __restrict__ B, long long ldb, void* __restrict__ out,
                                                       long long Mo, int No, long long K, long long kper) {
    constexpr int BK = IO == KFH_F32 ? 32 : 64, LDK = BK + 8, T = 64;
    constexpr int TILE = parts_of<IO>() * T * LDK;
    __shared__ __attribute__((aligned(16))) uint16_t smem[2 * TILE];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int wm = wave & 1, wn = wave >> 1;
    const long long m0 = (long long)blockIdx.x * T;
    const int n0 = blockIdx.y * T;
    const long long kb = (long long)blockIdx.z * kper, ke = min(kb + kper, K);
    f32x16 acc[1][1];
    zero_acc(acc);
    TileLoad<IO, AKC, T, BK> la;
    TileLoad<IO, BKC, T, BK> lb;
    for (long long k0 = kb; k0 < ke; k0 += BK) {
        la.load(A, lda, m0, Mo, k0, ke, tid);
        lb.load(B, ldb, n0, No, k0, ke, tid);
        __syncthreads();
        la.store(smem, tid); lb.store(smem + TILE, tid);
        __syncthreads();
        tile_mma<IO, 1, 1, T, T, BK>(smem, wm * 32, smem + TILE, wn * 32, lane, acc);
    }
    const long long m = m0 + wm * 32 + (lane & 31);
    if (m >= Mo) return;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const int n = n0 + wn * 32 + 8 * q + 4 * (lane >> 5);
        if (n >= No) continue;
        const f32x16& a = acc[0][0];
        if constexpr (SPLIT)
            store4<KFH_F32>(out, ((size_t)blockIdx.z * Mo + m) * No + n, a[4 * q], a[4 * q + 1], a[4 * q + 2], a[4 * q + 3]);
        else
            store4<IO>(out, (size_t)m * No + n, a[4 * q], a[4 * q + 1], a[4 * q + 2], a[4 * q + 3]);
    }
}

// out[i] = sum of `parts` fp32 values part[z * n + i], in order
__global__ __launch_bounds__(256) void ffn_sum_parts_kernel(const float* __restrict__ part, int parts, long long n,
                                                            void* __restrict__ out, int out_dtype) {
    const long long i = ((long long)blockIdx.x * 256 + threadIdx.x) * 4;
    if (i >= n) return;
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
    for (int z = 0; z < parts; ++z) {
        const f32x4 w = *reinterpret_cast<const f32x4*>(part + (size_t)z * n + i);
#pragma unroll
        for (int e = 0; e < 4; ++e) s[e] += w[e];
    }
    if (out_dtype == KFH_BF16) store4<KFH_BF16>(out, (size_t)i, s[0], s[1], s[2], s[3]);
    else store4<KFH_F32>(out, (size_t)i, s[0], s[1], s[2], s[3]);
}

// ---------------------------------------------------------------------------------------------
static size_t up256(size_t x) { return (x + 255) / 256 * 256; }

// ranges of rows the weight gradients are summed over in parallel: about 1024 workgroups, at least
// 256 rows each
static int wgrad_splits(long long M, long long tiles) {
    const long long want = max(1LL, 1024 / max(1LL, tiles)), most = max(1LL, (M + 255) / 256);
    return (int)min(min(want, most), 256LL);
}
static long long tiles64(long long a, long long b) { return ((a + 63) / 64) * ((b + 63) / 64); }
static size_t wgrad_part_bytes(long long M, int C, int F) {
    const size_t a = (size_t)wgrad_splits(M, tiles64(2 * F, C)) * 2 * F * C * 4;
    const size_t b = (size_t)wgrad_splits(M, tiles64(C, F)) * F * C * 4;
    return a > b ? a : b;
}

size_t gated_ffn_ws_bytes(long long M, int C, int F, int backward, int io_dtype) {
    const size_t e = io_dtype == KFH_F32 ? 4 : 2;
    if (!backward) return up256((size_t)M * F * e);
    return up256((size_t)M * F * e) + up256((size_t)M * 2 * F * e) + up256(wgrad_part_bytes(M, C, F));
}

template <int IO>
static void forward_t(const void* x, const void* w_in, const void* w_out, void* y, char* ws, long long M, int C, int F,
                      hipStream_t stream) {
    const dim3 block(256);
    hipLaunchKernelGGL((ffn_hidden_kernel<IO, false>), dim3((unsigned)((M + 63) / 64), (unsigned)((F + 63) / 64)), block, 0,
                       stream, x, nullptr, w_in, nullptr, ws, nullptr, M, C, F);
    hipLaunchKernelGGL((ffn_gemm_kernel<IO, true, true, false>), dim3((unsigned)((M + 63) / 64), (unsigned)((C + 63) / 64)),
                       block, 0, stream, ws, (long long)F, w_out, (long long)F, y, M, C, (long long)F, (long long)F);
}

template <int IO>
static void wgrad(const void* A, int Ma, const void* B, int Nb, float* part, void* out, int out_dtype, long long M,
                  hipStream_t stream) {
    const int splits = wgrad_splits(M, tiles64(Ma, Nb));
    long long per = (M + splits - 1) / splits;
    per = (per + 63) / 64 * 64;
    hipLaunchKernelGGL((ffn_gemm_kernel<IO, false, false, true>),
                       dim3((unsigned)((Ma + 63) / 64), (unsigned)((Nb + 63) / 64), (unsigned)splits), dim3(256), 0, stream, A,
                       (long long)Ma, B, (long long)Nb, part, (long long)Ma, Nb, M, per);
    const long long n = (long long)Ma * Nb;
    hipLaunchKernelGGL(ffn_sum_parts_kernel, dim3((unsigned)((n / 4 + 255) / 256)), dim3(256), 0, stream, part, splits, n,
                       out, out_dtype);
}

template <int IO>
static void backward_t(const void* dy, const void* x, const void* w_in, const void* w_out, void* dx, void* dw_in,
                       void* dw_out, int dw_dtype, char* ws, long long M, int C, int F, hipStream_t stream) {
    const size_t e = IO == KFH_F32 ? 4 : 2;
    char* h = ws;
    char* d = h + up256((size_t)M * F * e);
    float* part = reinterpret_cast<float*>(d + up256((size_t)M * 2 * F * e));
    const dim3 block(256);
    hipLaunchKernelGGL((ffn_hidden_kernel<IO, true>), dim3((unsigned)((M + 63) / 64), (unsigned)((F + 63) / 64)), block, 0,
                       stream, x, dy, w_in, w_out, h, d, M, C, F);
    // dy is read before dx, which may be written over it
    if (dw_out) wgrad<IO>(dy, C, h, F, part, dw_out, dw_dtype, M, stream);
    if (dw_in) wgrad<IO>(d, 2 * F, x, C, part, dw_in, dw_dtype, M, stream);
    if (dx)
        hipLaunchKernelGGL((ffn_gemm_kernel<IO, true, false, false>), dim3((unsigned)((M + 63) / 64), (unsigned)((C + 63) / 64)),
                           block, 0, stream, d, 2LL * F, w_in, (long long)C, dx, M, C, 2LL * F, 2LL * F);
}

void launch_gated_ffn_forward(const void* x, const void* w_in, const void* w_out, void* y, char* ws, long long M,
                              int C, int F, int io_dtype, hipStream_t stream) {
    if (io_dtype == KFH_F32) forward_t<KFH_F32>(x, w_in, w_out, y, ws, M, C, F, stream);
    else forward_t<KFH_BF16>(x, w_in, w_out, y, ws, M, C, F, stream);
}

void launch_gated_ffn_backward(const void* dy, const void* x, const void* w_in, const void* w_out, void* dx,
                               void* dw_in, void* dw_out, int dw_dtype, char* ws, long long M, int C, int F,
                               int io_dtype, hipStream_t stream) {
    if (io_dtype == KFH_F32) backward_t<KFH_F32>(dy, x, w_in, w_out, dx, dw_in, dw_out, dw_dtype, ws, M, C, F, stream);
    else backward_t<KFH_BF16>(dy, x, w_in, w_out, dx, dw_in, dw_out, dw_dtype, ws, M, C, F, stream);
}

}  // namespace kfh
