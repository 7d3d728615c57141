// Layer norm of [rows, C] tensors, forward and backward.
// Reference: src/kfold/model/primitives/normalization.py:61-91 (fp32 statistics, biased variance).
//
//   y = (x - mean) * rstd * gamma + beta,   rstd = (var + eps)^-1/2
//   with xh = (x - mean) * rstd and a = dy * gamma:
//   dx     = rstd * (a - mean_c(a) - xh * mean_c(a * xh))
//   dgamma = sum_rows dy * xh,   dbeta = sum_rows dy
//
// Statistics, row sums and a workgroup's sums over its rows are held in fp32; y and dx are rounded once, when
// they are stored.  The variance is taken from the deviations (two passes over the row), so a row far
// from zero loses no more than its mean's rounding.  The sums over rows go through per-workgroup partial sums that
// one more kernel adds in 64 bits, in a fixed order: the same call gives the same bits.
//
// Bound by memory traffic.  Up to 2048 channels every value is read once: 589824 x 256 bf16 forward 103 us
// (5.9 TB/s; a copy of 1 GiB, half of it writes, reaches 5.1), 147456 x 128 bf16 backward with the sums 25 us (21 + 4 for
// the partial sums; 114 MB).  Wider rows are read three times forward (the sum, the deviations, the result) and
// three times backward (the column sums, the row sums, dx): 16384 x 4096 bf16 1.3 TB/s
// forward, 1.5 backward (2048 channels: 5.0, 4.2).
// Widths that are no multiple of 8 go through single elements: 5001 x 765 fp32 backward 17 us (46 MB).
#include "train.hpp"

namespace kfh {

template <int IO>
__device__ __forceinline__ float ld1(const void* p, size_t i) {
    if constexpr (IO == KFH_BF16) return bf16_lo(static_cast<const uint16_t*>(p)[i]);
    else return static_cast<const float*>(p)[i];
}
template <int IO>
__device__ __forceinline__ void st1(void* p, size_t i, float v) {
    if constexpr (IO == KFH_BF16) static_cast<uint16_t*>(p)[i] = (uint16_t)pack_bf16(v, 0.f);
    else static_cast<float*>(p)[i] = v;
}

__device__ __forceinline__ float wave_sum64(float v) {
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) v += __shfl_xor(v, off);
    return v;
}

// ---- rows held in registers ---------------------------------------------------------------------
// LPR lanes share a row (64 / LPR rows per wavefront), each holding NJ * 8 of its values:
//   VEC : lane l holds the 16-byte-aligned groups of 8 channels l + LPR j (C % 8 == 0, 16-byte loads)
//   else: lane l holds the channels l + LPR i, i < 8 NJ (any width or alignment)
// so every value is read from memory once.  These kernels do nothing but stream: what they need is
// many bytes in flight, so a thread requests R rows before it uses the first.
template <int IO, bool VEC, int LPR, int NJ>
struct RegRow {
    static __device__ __forceinline__ int chan(int l, int i) {
        return VEC ? 8 * (l + LPR * (i >> 3)) + (i & 7) : l + LPR * i;
    }
    // A row as it comes from memory.  All rows of a step are fetched, then expanded behind a scheduling
    // barrier: left to itself the compiler waits for 2-byte loads one by one to save registers (measured
    // at 65536 x 765 bf16: 410 us for the backward pass instead of 82).
    struct Raw {
        u32x4 q[VEC ? NJ * (IO == KFH_BF16 ? 1 : 2) : 1];
        uint32_t w[VEC ? 1 : NJ * 8];
    };
    // no branch on the channel: a lane behind the row reads the row's end, and `trim` clears what it got
    static __device__ __forceinline__ void fetch(const void* p, size_t base, int C, int l, Raw& raw) {
        if constexpr (VEC) {
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                const size_t e = base + min(8 * (l + LPR * j), C - 8);
                if constexpr (IO == KFH_BF16) {
                    raw.q[j] = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(p) + e);
                } else {
                    const u32x4* s = reinterpret_cast<const u32x4*>(static_cast<const float*>(p) + e);
                    raw.q[2 * j] = s[0];
                    raw.q[2 * j + 1] = s[1];
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8 * NJ; ++i) {
                const size_t e = base + min(l + LPR * i, C - 1);
                if constexpr (IO == KFH_BF16) raw.w[i] = static_cast<const uint16_t*>(p)[e];
                else raw.w[i] = static_cast<const uint32_t*>(p)[e];
            }
        }
    }
    static __device__ __forceinline__ void expand(const Raw& raw, float (&v)[NJ * 8]) {
#pragma unroll
        for (int i = 0; i < 8 * NJ; ++i) {
            if constexpr (VEC && IO == KFH_BF16) v[i] = (i & 1) ? bf16_hi(raw.q[i >> 3][(i & 7) >> 1]) : bf16_lo(raw.q[i >> 3][(i & 7) >> 1]);
            else if constexpr (VEC) v[i] = __uint_as_float(raw.q[i >> 2][i & 3]);
            else v[i] = __uint_as_float(IO == KFH_BF16 ? raw.w[i] << 16 : raw.w[i]);
        }
    }
    static __device__ __forceinline__ void trim(int C, int l, float (&v)[NJ * 8]) {
#pragma unroll
        for (int i = 0; i < 8 * NJ; ++i)
            if (chan(l, i) >= C) v[i] = 0.f;
    }
    // gamma or beta of this lane's channels
    static __device__ __forceinline__ void params(const float* p, float none, int C, int l, float (&v)[NJ * 8]) {
        if (p) {
            typename RegRow<KFH_F32, VEC, LPR, NJ>::Raw raw;
            RegRow<KFH_F32, VEC, LPR, NJ>::fetch(p, 0, C, l, raw);
            RegRow<KFH_F32, VEC, LPR, NJ>::expand(raw, v);
        } else {
#pragma unroll
            for (int i = 0; i < 8 * NJ; ++i) v[i] = none;
        }
    }
    static __device__ __forceinline__ void store(void* p, size_t base, int C, int l, const float (&v)[NJ * 8]) {
        if constexpr (VEC) {
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                const int c = 8 * (l + LPR * j);
                if (c >= C) continue;
                if constexpr (IO == KFH_BF16) {
                    u32x4 w;
#pragma unroll
                    for (int e = 0; e < 4; ++e) w[e] = pack_bf16(v[8 * j + 2 * e], v[8 * j + 2 * e + 1]);
                    *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(p) + base + c) = w;
                } else {
                    f32x4* d = reinterpret_cast<f32x4*>(static_cast<float*>(p) + base + c);
                    d[0] = f32x4{v[8 * j], v[8 * j + 1], v[8 * j + 2], v[8 * j + 3]};
                    d[1] = f32x4{v[8 * j + 4], v[8 * j + 5], v[8 * j + 6], v[8 * j + 7]};
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8 * NJ; ++i)
                if (l + LPR * i < C) st1<IO>(p, base + l + LPR * i, v[i]);
        }
    }
    // sums over the LPR lanes of a row, the rows' steps side by side
    template <int R>
    static __device__ __forceinline__ void sum(float (&s)[R]) {
#pragma unroll
        for (int off = 1; off < LPR; off <<= 1) {
            float o[R];
#pragma unroll
            for (int k = 0; k < R; ++k) o[k] = __shfl_xor(s[k], off);
#pragma unroll
            for (int k = 0; k < R; ++k) s[k] += o[k];
        }
    }
};

template <int IO, bool VEC, int LPR, int NJ, int R>
__global__ __launch_bounds__(256) void ln_fwd_reg_kernel(const void* x, const float* __restrict__ gamma,
                                                         const float* __restrict__ beta, void* y,
                                                         float* __restrict__ mean_out, float* __restrict__ rstd_out,
                                                         long long M, int C, float eps) {
    using Row = RegRow<IO, VEC, LPR, NJ>;
    constexpr int N = NJ * 8, RPB = 256 / LPR;              // rows side by side in the workgroup
    const int l = threadIdx.x % LPR, g = threadIdx.x / LPR;
    // divided by, not multiplied with a rounded 1 / C: a row of one value gives exactly 0 where its sum is exact, as
    // with bf16 values (8 bits, at most 2048 of them)
    const float fc = (float)C;
    float gam[N], bet[N];
    Row::params(gamma, 1.f, C, l, gam);
    Row::params(beta, 0.f, C, l, bet);
    for (long long r0 = (long long)blockIdx.x * RPB * R + g; r0 - g < M; r0 += (long long)gridDim.x * RPB * R) {
        float v[R][N], mean[R], q[R];
        typename Row::Raw raw[R];
#pragma unroll
        for (int k = 0; k < R; ++k) Row::fetch(x, (size_t)min(r0 + k * RPB, M - 1) * C, C, l, raw[k]);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int k = 0; k < R; ++k) {
            Row::expand(raw[k], v[k]);
            Row::trim(C, l, v[k]);
            mean[k] = 0.f;
#pragma unroll
            for (int i = 0; i < N; ++i) mean[k] += v[k][i];
        }
        Row::sum(mean);
#pragma unroll
        for (int k = 0; k < R; ++k) {
            mean[k] /= fc;
            q[k] = 0.f;
#pragma unroll
            for (int i = 0; i < N; ++i) v[k][i] -= mean[k];
            Row::trim(C, l, v[k]);
#pragma unroll
            for (int i = 0; i < N; ++i) q[k] += v[k][i] * v[k][i];
        }
        Row::sum(q);
#pragma unroll
        for (int k = 0; k < R; ++k) {
            const long long r = r0 + k * RPB;
            const float rstd = 1.0f / sqrtf(q[k] / fc + eps);
#pragma unroll
            for (int i = 0; i < N; ++i) v[k][i] = v[k][i] * rstd * gam[i] + bet[i];
            if (r < M) {
                Row::store(y, (size_t)r * C, C, l, v[k]);
                if (mean_out && l == 0) { mean_out[r] = mean[k]; rstd_out[r] = rstd; }
            }
        }
    }
}

// dx and, with SUMS, this workgroup's share of dgamma and dbeta: a lane adds up its channels over the
// rows it sees, then the lanes and wavefronts that share a channel are added through LDS in a fixed
// order; part[blockIdx.x] = { dgamma [C], dbeta [C] }.
template <int IO, bool VEC, int LPR, int NJ, int R, bool SUMS>
__global__ __launch_bounds__(256) void ln_bwd_reg_kernel(const void* dy, const void* __restrict__ x,
                                                         const float* __restrict__ mean_in,
                                                         const float* __restrict__ rstd_in,
                                                         const float* __restrict__ gamma, void* dx,
                                                         float* __restrict__ part, long long M, int C) {
    using Row = RegRow<IO, VEC, LPR, NJ>;
    constexpr int N = NJ * 8, RPB = 256 / LPR;
    const int l = threadIdx.x % LPR, g = threadIdx.x / LPR;
    const float inv = 1.0f / C;
    float gam[N], dg[N], db[N];
    Row::params(gamma, 1.f, C, l, gam);
#pragma unroll
    for (int i = 0; i < N; ++i) dg[i] = db[i] = 0.f;
    for (long long r0 = (long long)blockIdx.x * RPB * R + g; r0 - g < M; r0 += (long long)gridDim.x * RPB * R) {
        float a[R][N], v[R][N], mean[R], rstd[R], s1[R], s2[R];
        typename Row::Raw rawa[R], rawv[R];
#pragma unroll
        for (int k = 0; k < R; ++k) {
            const long long r = min(r0 + k * RPB, M - 1);
            Row::fetch(dy, (size_t)r * C, C, l, rawa[k]);
            Row::fetch(x, (size_t)r * C, C, l, rawv[k]);
            mean[k] = mean_in[r];
            rstd[k] = rstd_in[r];
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int k = 0; k < R; ++k) {
            Row::expand(rawa[k], a[k]);
            Row::expand(rawv[k], v[k]);
            s1[k] = s2[k] = 0.f;
#pragma unroll
            for (int i = 0; i < N; ++i) v[k][i] = (v[k][i] - mean[k]) * rstd[k];
            Row::trim(C, l, v[k]);
            if (SUMS && r0 + k * RPB < M) {
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    dg[i] += a[k][i] * v[k][i];
                    db[i] += a[k][i];
                }
            }
#pragma unroll
            for (int i = 0; i < N; ++i) a[k][i] *= gam[i];
            Row::trim(C, l, a[k]);           // (the product: 0 times an infinite weight would be NaN)
#pragma unroll
            for (int i = 0; i < N; ++i) {
                s1[k] += a[k][i];
                s2[k] += a[k][i] * v[k][i];
            }
        }
        if (dx) {
            Row::sum(s1);
            Row::sum(s2);
#pragma unroll
            for (int k = 0; k < R; ++k) {
                const long long r = r0 + k * RPB;
                const float m1 = s1[k] * inv, m2 = s2[k] * inv;
#pragma unroll
                for (int i = 0; i < N; ++i) a[k][i] = rstd[k] * (a[k][i] - m1 - v[k][i] * m2);
                if (r < M) Row::store(dx, (size_t)r * C, C, l, a[k]);
            }
        }
    }
    if constexpr (SUMS) {
        // lanes of one wavefront that hold the same channels
#pragma unroll
        for (int off = LPR; off < 64; off <<= 1)
#pragma unroll
            for (int i = 0; i < N; ++i) {
                dg[i] += __shfl_xor(dg[i], off);
                db[i] += __shfl_xor(db[i], off);
            }
        // the four wavefronts
        __shared__ float red[4][N * LPR];
        const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
        for (int which = 0; which < 2; ++which) {
            if (lane < LPR)
#pragma unroll
                for (int i = 0; i < N; ++i) red[wave][i * LPR + lane] = which ? db[i] : dg[i];
            __syncthreads();
            for (int k = threadIdx.x; k < N * LPR; k += 256) {
                const int c = Row::chan(k % LPR, k / LPR);
                if (c < C)
                    part[((size_t)blockIdx.x * 2 + which) * C + c] = (red[0][k] + red[1][k]) + (red[2][k] + red[3][k]);
            }
            __syncthreads();
        }
    }
}

// ---- rows too wide for registers: one wavefront per row ----------------------------------------
// Element c of the row belongs to lane c % 64 in every pass, so y may be written over x.
template <int IO>
__global__ __launch_bounds__(256) void ln_fwd_any_kernel(const void* x, const float* __restrict__ gamma,
                                                         const float* __restrict__ beta, void* y,
                                                         float* __restrict__ mean_out, float* __restrict__ rstd_out,
                                                         long long M, int C, float eps) {
    const int lane = threadIdx.x & 63;
    for (long long r = (long long)blockIdx.x * 4 + (threadIdx.x >> 6); r < M; r += (long long)gridDim.x * 4) {
        const size_t base = (size_t)r * C;
        float s = 0.f;
        for (int c = lane; c < C; c += 64) s += ld1<IO>(x, base + c);
        const float mean = wave_sum64(s) / C;
        float q = 0.f;
        for (int c = lane; c < C; c += 64) { const float d = ld1<IO>(x, base + c) - mean; q += d * d; }
        const float rstd = 1.0f / sqrtf(wave_sum64(q) / C + eps);
        for (int c = lane; c < C; c += 64) {
            float v = (ld1<IO>(x, base + c) - mean) * rstd;
            if (gamma) v *= gamma[c];
            if (beta) v += beta[c];
            st1<IO>(y, base + c, v);
        }
        if (mean_out && lane == 0) { mean_out[r] = mean; rstd_out[r] = rstd; }
    }
}

template <int IO>
__global__ __launch_bounds__(256) void ln_bwd_dx_any_kernel(const void* dy, const void* __restrict__ x,
                                                            const float* __restrict__ mean_in,
                                                            const float* __restrict__ rstd_in,
                                                            const float* __restrict__ gamma, void* dx, long long M,
                                                            int C) {
    const int lane = threadIdx.x & 63;
    for (long long r = (long long)blockIdx.x * 4 + (threadIdx.x >> 6); r < M; r += (long long)gridDim.x * 4) {
        const size_t base = (size_t)r * C;
        const float mean = mean_in[r], rstd = rstd_in[r];
        float s1 = 0.f, s2 = 0.f;
        for (int c = lane; c < C; c += 64) {
            const float a = ld1<IO>(dy, base + c) * (gamma ? gamma[c] : 1.f);
            s1 += a;
            s2 += a * ((ld1<IO>(x, base + c) - mean) * rstd);
        }
        s1 = wave_sum64(s1) / C;
        s2 = wave_sum64(s2) / C;
        for (int c = lane; c < C; c += 64) {
            const float a = ld1<IO>(dy, base + c) * (gamma ? gamma[c] : 1.f);
            const float xh = (ld1<IO>(x, base + c) - mean) * rstd;
            st1<IO>(dx, base + c, rstd * (a - s1 - xh * s2));
        }
    }
}

// Partial sums over rows [blockIdx.y * rows_per, ...) of 64 columns: a lane owns a column, the four
// wavefronts take every fourth row; part[blockIdx.y] = { dgamma [C], dbeta [C] }.
template <int IO>
__global__ __launch_bounds__(256) void ln_bwd_cols_any_kernel(const void* __restrict__ dy, const void* __restrict__ x,
                                                              const float* __restrict__ mean_in,
                                                              const float* __restrict__ rstd_in,
                                                              float* __restrict__ part, long long M, int C,
                                                              long long rows_per) {
    __shared__ float red[2][4][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int c = blockIdx.x * 64 + lane;
    const long long r0 = (long long)blockIdx.y * rows_per, r1 = min(r0 + rows_per, M);
    float g = 0.f, b = 0.f;
    if (c < C) {
        for (long long r = r0 + wave; r < r1; r += 4) {
            const float d = ld1<IO>(dy, (size_t)r * C + c);
            g += d * ((ld1<IO>(x, (size_t)r * C + c) - mean_in[r]) * rstd_in[r]);
            b += d;
        }
    }
    red[0][wave][lane] = g;
    red[1][wave][lane] = b;
    __syncthreads();
    if (wave < 2 && c < C) {
        const float(*p)[64] = red[wave];
        part[((size_t)blockIdx.y * 2 + wave) * C + c] = (p[0][lane] + p[1][lane]) + (p[2][lane] + p[3][lane]);
    }
}

// dgamma / dbeta <- sums of nblk partial rows of 2C values: 32 columns per workgroup, 32 strided
// groups of partial rows, added in a fixed order.  In 64 bits: a few additions more per result, and the
// error is that of the partial sums alone (db of 5001 rows: 1.3e-7 of its norm in 32 bits).
__global__ __launch_bounds__(1024) void ln_bwd_finish_kernel(const float* __restrict__ part, int nblk, int C,
                                                             float* __restrict__ dgamma, float* __restrict__ dbeta) {
    __shared__ double red[32][32];
    const int col = threadIdx.x & 31, grp = threadIdx.x >> 5;
    const int c = blockIdx.x * 32 + col;
    double s = 0.;
    if (c < 2 * C) {
#pragma unroll 8
        for (int i = grp; i < nblk; i += 32) s += part[(size_t)i * 2 * C + c];
    }
    red[grp][col] = s;
    __syncthreads();
    if (grp == 0 && c < 2 * C) {
        s = 0.;
#pragma unroll
        for (int k = 0; k < 32; ++k) s += red[k][col];
        if (c < C) { if (dgamma) dgamma[c] = (float)s; }
        else if (dbeta) dbeta[c - C] = (float)s;
    }
}

// Rows per register kernel: lanes per row and groups of 8 values per lane by the width, so that a
// row is spread over as few lanes as hold it in at most 8 (up to 512 channels), then 64 lanes.
// f(LPR, NJ as integral constants) is called for the shape; false if the width has none.
template <int V> struct Int { static constexpr int v = V; };
template <class F>
static bool by_width(int C, F f) {
    if (C <= 64) f(Int<8>{}, Int<1>{});
    else if (C <= 128) f(Int<16>{}, Int<1>{});
    else if (C <= 256) f(Int<32>{}, Int<1>{});
    else if (C <= 512) f(Int<64>{}, Int<1>{});
    else if (C <= 1024) f(Int<64>{}, Int<2>{});
    else if (C <= 2048) f(Int<64>{}, Int<4>{});
    else return false;
    return true;
}

// workgroups for M rows of which one takes `rows` at a time; beyond 2^20 of them a workgroup takes several turns
static unsigned row_grid(long long M, long long rows) { return (unsigned)min((M + rows - 1) / rows, 1LL << 20); }
static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// partial rows of a backward call: enough workgroups to fill the chip with a few each, and enough rows
// per workgroup (16) that the partial sums stay small beside the rows
int ln_bwd_blocks(long long M) {
    return (int)max(1LL, min((M + 15) / 16, 1024LL));
}

template <int IO>
static void ln_forward_t(const void* x, const float* gamma, const float* beta, void* y, float* mean, float* rstd,
                         long long M, int C, float eps, hipStream_t stream) {
    const dim3 block(256);
    const bool vec = C % 8 == 0 && aligned16(x) && aligned16(y) && aligned16(gamma) && aligned16(beta);
    const bool done = by_width(C, [&](auto lpr, auto nj) {
        constexpr int LPR = decltype(lpr)::v, NJ = decltype(nj)::v, R = NJ == 1 ? 4 : NJ == 2 ? 2 : 1;
        const dim3 grid(row_grid(M, (long long)(256 / LPR) * R));
        if (vec)
            hipLaunchKernelGGL((ln_fwd_reg_kernel<IO, true, LPR, NJ, R>), grid, block, 0, stream, x, gamma, beta, y, mean,
                               rstd, M, C, eps);
        else
            hipLaunchKernelGGL((ln_fwd_reg_kernel<IO, false, LPR, NJ, R>), grid, block, 0, stream, x, gamma, beta, y, mean,
                               rstd, M, C, eps);
    });
    if (!done)
        hipLaunchKernelGGL(ln_fwd_any_kernel<IO>, dim3(row_grid(M, 4)), block, 0, stream, x, gamma, beta, y, mean, rstd, M,
                           C, eps);
}

void launch_ln_forward(const void* x, int io_dtype, const float* gamma, const float* beta, void* y, float* mean,
                       float* rstd, long long M, int C, float eps, hipStream_t stream) {
    if (io_dtype == KFH_F32) ln_forward_t<KFH_F32>(x, gamma, beta, y, mean, rstd, M, C, eps, stream);
    else ln_forward_t<KFH_BF16>(x, gamma, beta, y, mean, rstd, M, C, eps, stream);
}

template <int IO>
static void ln_backward_t(const void* dy, const void* x, const float* mean, const float* rstd, const float* gamma,
                          void* dx, float* dgamma, float* dbeta, float* part, long long M, int C, hipStream_t stream) {
    const dim3 block(256);
    const bool sums = dgamma || dbeta;
    const int nblk = ln_bwd_blocks(M);
    const bool vec = C % 8 == 0 && aligned16(x) && aligned16(dy) && aligned16(dx) && aligned16(gamma);
    const bool done = by_width(C, [&](auto lpr, auto nj) {
        constexpr int LPR = decltype(lpr)::v, NJ = decltype(nj)::v, R = NJ == 1 ? 2 : 1;
        const dim3 grid(sums ? (unsigned)nblk : row_grid(M, (long long)(256 / LPR) * R));
#define KFH_LN_BWD(VEC, SUMS)                                                                                        \
    hipLaunchKernelGGL((ln_bwd_reg_kernel<IO, VEC, LPR, NJ, R, SUMS>), grid, block, 0, stream, dy, x, mean, rstd, gamma, \
                       dx, part, M, C)
        if (vec) { if (sums) KFH_LN_BWD(true, true); else KFH_LN_BWD(true, false); }
        else { if (sums) KFH_LN_BWD(false, true); else KFH_LN_BWD(false, false); }
#undef KFH_LN_BWD
    });
    if (!done && sums)                       // the column sums read dy, which dx may overwrite: they come first
        hipLaunchKernelGGL(ln_bwd_cols_any_kernel<IO>, dim3((unsigned)((C + 63) / 64), (unsigned)nblk), block, 0, stream, dy,
                           x, mean, rstd, part, M, C, (M + nblk - 1) / nblk);
    if (sums)
        hipLaunchKernelGGL(ln_bwd_finish_kernel, dim3((unsigned)((2 * C + 31) / 32)), dim3(1024), 0, stream, part, nblk, C,
                           dgamma, dbeta);
    if (!done && dx)
        hipLaunchKernelGGL(ln_bwd_dx_any_kernel<IO>, dim3(row_grid(M, 4)), block, 0, stream, dy, x, mean, rstd, gamma, dx, M,
                           C);
}

void launch_ln_backward(const void* dy, const void* x, int io_dtype, const float* mean, const float* rstd,
                        const float* gamma, void* dx, float* dgamma, float* dbeta, float* part, long long M, int C,
                        hipStream_t stream) {
    if (M == 0) {                            // sums over no rows
        hipLaunchKernelGGL(ln_bwd_finish_kernel, dim3((unsigned)((2 * C + 31) / 32)), dim3(1024), 0, stream, part, 0, C,
                           dgamma, dbeta);
        return;
    }
    if (io_dtype == KFH_F32) ln_backward_t<KFH_F32>(dy, x, mean, rstd, gamma, dx, dgamma, dbeta, part, M, C, stream);
    else ln_backward_t<KFH_BF16>(dy, x, mean, rstd, gamma, dx, dgamma, dbeta, part, M, C, stream);
}

}  // namespace kfh
