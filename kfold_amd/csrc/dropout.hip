// Dropout whose mask is computed where it is needed and never stored:
//     y = [residual +] (keep ? x * scale : 0),   keep(i) = r16(i) >= t,
//     t = round(p * 2^16),   scale = 2^16 / (2^16 - t)
// The mask index i runs over x's shape [outer, shared, inner] without the shared dimension (one
// value covers all `shared` positions: row-wise / column-wise dropout of the pair track).  r16(i) is
// half-word i % 8 (low half of a word first) of the four words that Philox4x32-10 (Salmon, Moraes,
// Dror, Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC 2011) gives for the counter
// (i / 8 in words 0-1, offset in words 2-3) under the 64-bit key `seed`.  Sixteen random bits per
// element keep the generator at 1/8 call per element; the drop probability is a multiple of 2^-16
// and the scale uses the same multiple, so the expectation of y is exact.  The gradient is the same
// map applied to dy.  Dropped values are never multiplied: inf and NaN there leave 0.
// The product and the sum are fp32, rounded once.
#include "train.hpp"

namespace kfh {

struct Philox { uint32_t w[4]; };

__device__ __forceinline__ Philox philox10(uint64_t ctr, uint64_t offset, uint64_t seed) {
    uint32_t c0 = (uint32_t)ctr, c1 = (uint32_t)(ctr >> 32), c2 = (uint32_t)offset, c3 = (uint32_t)(offset >> 32);
    uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const uint64_t a = (uint64_t)0xD2511F53u * c0, b = (uint64_t)0xCD9E8D57u * c2;
        c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
        c1 = (uint32_t)b;
        c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
        c3 = (uint32_t)a;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return Philox{{c0, c1, c2, c3}};
}

template <int IO>
__device__ __forceinline__ void drop1(const DropArgs& p, size_t e, bool keep) {
    float v = 0.f;
    if constexpr (IO == KFH_BF16) {
        if (keep) v = bf16_lo(static_cast<const uint16_t*>(p.x)[e]) * p.scale;
        if (p.residual) v += bf16_lo(static_cast<const uint16_t*>(p.residual)[e]);
        static_cast<uint16_t*>(p.y)[e] = (uint16_t)pack_bf16(v, 0.f);
    } else {
        if (keep) v = static_cast<const float*>(p.x)[e] * p.scale;
        if (p.residual) v += static_cast<const float*>(p.residual)[e];
        static_cast<float*>(p.y)[e] = v;
    }
}

// any shape and alignment: a thread owns 8 consecutive mask values (one generator call) and, with
// blockIdx.y, every gridDim.y-th of the shared positions they cover
template <int IO>
__global__ __launch_bounds__(256) void dropout_any_kernel(DropArgs p) {
    const long long n = p.outer * p.inner;
    const long long g = (long long)blockIdx.x * 256 + threadIdx.x;
    if (g * 8 >= n) return;
    const Philox r = philox10((uint64_t)g, p.offset, p.seed_dev ? *p.seed_dev : p.seed);
    for (int j = 0; j < 8; ++j) {
        const long long i = g * 8 + j;
        if (i >= n) return;
        const bool keep = ((r.w[j >> 1] >> (16 * (j & 1))) & 0xffffu) >= p.t;
        const long long o = i / p.inner, c = i % p.inner;
        for (long long s = blockIdx.y; s < p.shared; s += gridDim.y)
            drop1<IO>(p, (size_t)((o * p.shared + s) * p.inner + c), keep);
    }
}

void launch_dropout(const DropArgs& p, int io_dtype, hipStream_t stream) {
    const long long groups = (p.outer * p.inner + 7) / 8;
    const dim3 grid((unsigned)((groups + 255) / 256), (unsigned)min(p.shared, 1024LL)), block(256);
    if (io_dtype == KFH_F32)
        hipLaunchKernelGGL(dropout_any_kernel<KFH_F32>, grid, block, 0, stream, p);
    else
        hipLaunchKernelGGL(dropout_any_kernel<KFH_BF16>, grid, block, 0, stream, p);
}

}  // namespace kfh
