// Layer norm of [rows, C] tensors, forward and backward.
// Reference: src/kfold/model/primitives/normalization.py:61-91 (fp32 statistics, biased variance).
//
//   y = (x - mean) * rstd * gamma + beta,   rstd = (var + eps)^-1/2
//   with xh = (x - mean) * rstd and a = dy * gamma:
//   dx     = rstd * (a - mean_c(a) - xh * mean_c(a * xh))
//   dgamma = sum_rows dy * xh,   dbeta = sum_rows dy
//
// Statistics, row sums and the sums over rows are held in fp32; y and dx are rounded once, when they
// are stored.  The variance is taken from the deviations (two passes over the row), so a row far
// from zero loses nothing.  The sums over rows go through per-workgroup partial sums that one more
// kernel adds in a fixed order: the same call gives the same bits.
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

// ---- any width, any alignment: one wavefront per row ------------------------------------------
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

// dgamma / dbeta <- sums of nblk partial rows of 2C values: 32 columns per workgroup, 8 strided
// groups of partial rows, added in a fixed order.
__global__ __launch_bounds__(256) void ln_bwd_finish_kernel(const float* __restrict__ part, int nblk, int C,
                                                            float* __restrict__ dgamma, float* __restrict__ dbeta) {
    __shared__ float red[8][32];
    const int col = threadIdx.x & 31, grp = threadIdx.x >> 5;
    const int c = blockIdx.x * 32 + col;
    float s = 0.f;
    if (c < 2 * C)
        for (int i = grp; i < nblk; i += 8) s += part[(size_t)i * 2 * C + c];
    red[grp][col] = s;
    __syncthreads();
    if (grp == 0 && c < 2 * C) {
        s = ((red[0][col] + red[1][col]) + (red[2][col] + red[3][col])) +
            ((red[4][col] + red[5][col]) + (red[6][col] + red[7][col]));
        if (c < C) { if (dgamma) dgamma[c] = s; }
        else if (dbeta) dbeta[c - C] = s;
    }
}

// partial rows of a backward call: enough workgroups to fill the chip, at least 64 rows each
int ln_bwd_blocks(long long M, int C) {
    (void)C;
    return (int)max(1LL, min((M + 63) / 64, 512LL));
}

// workgroups of four rows each; beyond 2^20 of them a workgroup takes several
static unsigned row_grid(long long M) { return (unsigned)min((M + 3) / 4, 1LL << 20); }

void launch_ln_forward(const void* x, int io_dtype, const float* gamma, const float* beta, void* y, float* mean,
                       float* rstd, long long M, int C, float eps, hipStream_t stream) {
    const dim3 grid(row_grid(M)), block(256);
    if (io_dtype == KFH_F32)
        hipLaunchKernelGGL(ln_fwd_any_kernel<KFH_F32>, grid, block, 0, stream, x, gamma, beta, y, mean, rstd, M, C, eps);
    else
        hipLaunchKernelGGL(ln_fwd_any_kernel<KFH_BF16>, grid, block, 0, stream, x, gamma, beta, y, mean, rstd, M, C, eps);
}

void launch_ln_backward(const void* dy, const void* x, int io_dtype, const float* mean, const float* rstd,
                        const float* gamma, void* dx, float* dgamma, float* dbeta, float* part, long long M, int C,
                        hipStream_t stream) {
    const dim3 block(256);
    if (M == 0) {                            // sums over no rows
        hipLaunchKernelGGL(ln_bwd_finish_kernel, dim3((unsigned)((2 * C + 31) / 32)), block, 0, stream, part, 0, C, dgamma,
                           dbeta);
        return;
    }
    const int nblk = ln_bwd_blocks(M, C);
    // the column sums read dy, which dx may overwrite: they come first
    if (dgamma || dbeta) {
        const dim3 cgrid((unsigned)((C + 63) / 64), (unsigned)nblk);
        const long long per = (M + nblk - 1) / nblk;
        if (io_dtype == KFH_F32)
            hipLaunchKernelGGL(ln_bwd_cols_any_kernel<KFH_F32>, cgrid, block, 0, stream, dy, x, mean, rstd, part, M, C, per);
        else
            hipLaunchKernelGGL(ln_bwd_cols_any_kernel<KFH_BF16>, cgrid, block, 0, stream, dy, x, mean, rstd, part, M, C, per);
        hipLaunchKernelGGL(ln_bwd_finish_kernel, dim3((unsigned)((2 * C + 31) / 32)), block, 0, stream, part, nblk, C,
                           dgamma, dbeta);
    }
    if (dx) {
        const dim3 grid(row_grid(M));
        if (io_dtype == KFH_F32)
            hipLaunchKernelGGL(ln_bwd_dx_any_kernel<KFH_F32>, grid, block, 0, stream, dy, x, mean, rstd, gamma, dx, M, C);
        else
            hipLaunchKernelGGL(ln_bwd_dx_any_kernel<KFH_BF16>, grid, block, 0, stream, dy, x, mean, rstd, gamma, dx, M, C);
    }
}

}  // namespace kfh
