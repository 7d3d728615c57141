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
//
// Bound by memory traffic, the generator (about 60 VALU instructions per call) beside it: 768 x 768 x 128 bf16
// row-wise with residual 86 us (453 MB, 5.3 TB/s), 32.9 M fp32 with a mask value each 48.5 us (263 MB, 5.4 TB/s) where
// inputs and outputs change from call to call (a copy of them takes 50), 40 us on the same tensors again and again,
// which the 256 MB last-level cache then holds in part.
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

template <int IO> struct Vals8;               // 8 consecutive values as they come from memory
template <> struct Vals8<KFH_BF16> { u32x4 w; };
template <> struct Vals8<KFH_F32> { f32x4 a, b; };

template <int IO>
__device__ __forceinline__ void ld8(const void* p, size_t e, Vals8<IO>& v) {
    if constexpr (IO == KFH_BF16) v.w = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(p) + e);
    else {
        const f32x4* q = reinterpret_cast<const f32x4*>(static_cast<const float*>(p) + e);
        v.a = q[0];
        v.b = q[1];
    }
}
template <int IO>
__device__ __forceinline__ float val(const Vals8<IO>& v, int j) {
    if constexpr (IO == KFH_BF16) return (j & 1) ? bf16_hi(v.w[j >> 1]) : bf16_lo(v.w[j >> 1]);
    else return j < 4 ? v.a[j & 3] : v.b[j & 3];
}

// y[e .. e+7] = [residual +] (keep ? x * scale : 0); bit j of `keep`: element e + j
template <int IO>
__device__ __forceinline__ void drop8(const DropArgs& p, size_t e, unsigned keep, const Vals8<IO>& x, const Vals8<IO>& r) {
    float o[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        o[j] = (keep >> j) & 1 ? val<IO>(x, j) * p.scale : 0.f;
        if (p.residual) o[j] += val<IO>(r, j);
    }
    if constexpr (IO == KFH_BF16) {
        *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(p.y) + e) =
            u32x4{pack_bf16(o[0], o[1]), pack_bf16(o[2], o[3]), pack_bf16(o[4], o[5]), pack_bf16(o[6], o[7])};
    } else {
        f32x4* d = reinterpret_cast<f32x4*>(static_cast<float*>(p.y) + e);
        d[0] = f32x4{o[0], o[1], o[2], o[3]};
        d[1] = f32x4{o[4], o[5], o[6], o[7]};
    }
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

__device__ __forceinline__ unsigned keep_bits(const Philox& r, uint32_t t) {
    unsigned k = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) k |= (unsigned)(((r.w[j >> 1] >> (16 * (j & 1))) & 0xffffu) >= t) << j;
    return k;
}

// Any shape: a thread takes 8 consecutive elements.  Without a shared dimension those are one
// generator call; with one, their mask indices follow the row they lie in and the generator is called
// again where they leave a group of 8.  VEC: x, residual and y at 16-byte boundaries.
template <int IO, bool VEC, bool SHARED>
__global__ __launch_bounds__(256) void dropout_flat_kernel(DropArgs p) {
    const long long n = p.outer * p.shared * p.inner;
    const long long g = (long long)blockIdx.x * 256 + threadIdx.x;
    const long long e0 = g * 8;
    if (e0 >= n) return;
    const bool whole = VEC && e0 + 8 <= n;
    Vals8<IO> x, r;
    if (whole) {                              // the values travel while the generator runs
        ld8<IO>(p.x, (size_t)e0, x);
        if (p.residual) ld8<IO>(p.residual, (size_t)e0, r);
    }
    const unsigned long long seed = p.seed_dev ? *p.seed_dev : p.seed;
    unsigned keep;
    if constexpr (!SHARED) {
        keep = keep_bits(philox10((uint64_t)g, p.offset, seed), p.t);
    } else {
        const long long row = e0 / p.inner;
        long long o = row / p.shared, s = row - o * p.shared, c = e0 - row * p.inner, at = -1;
        unsigned bits = 0;
        keep = 0;
#pragma unroll 1
        for (int j = 0; j < 8; ++j) {
            const long long i = o * p.inner + c;
            if ((i >> 3) != at) {
                at = i >> 3;
                bits = keep_bits(philox10((uint64_t)at, p.offset, seed), p.t);
            }
            keep |= ((bits >> (i & 7)) & 1u) << j;
            if (++c == p.inner) {
                c = 0;
                if (++s == p.shared) { s = 0; ++o; }
            }
        }
    }
    if (whole) {
        drop8<IO>(p, (size_t)e0, keep, x, r);
    } else {
        for (int j = 0; j < 8 && e0 + j < n; ++j) drop1<IO>(p, (size_t)(e0 + j), (keep >> j) & 1);
    }
}

// A shared dimension with rows of a multiple of 8 values at 16-byte boundaries: a thread draws the
// mask of 8 values once and takes them through the shared positions [blockIdx.y * per, + per), U of
// them requested at a time.
template <int IO, int U>
__global__ __launch_bounds__(256) void dropout_shared_kernel(DropArgs p, int per) {
    const long long g = (long long)blockIdx.x * 256 + threadIdx.x, c8 = p.inner >> 3;
    if (g >= p.outer * c8) return;
    const long long o = g / c8, c = (g - o * c8) * 8;
    const unsigned keep = keep_bits(philox10((uint64_t)g, p.offset, p.seed_dev ? *p.seed_dev : p.seed), p.t);
    const long long s0 = (long long)blockIdx.y * per, s1 = min(s0 + per, p.shared);
    for (long long s = s0; s < s1; s += U) {
        Vals8<IO> x[U], r[U];
        size_t e[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            e[u] = (size_t)((o * p.shared + min(s + u, s1 - 1)) * p.inner + c);
            ld8<IO>(p.x, e[u], x[u]);
            if (p.residual) ld8<IO>(p.residual, e[u], r[u]);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (s + u < s1) drop8<IO>(p, e[u], keep, x[u], r[u]);
    }
}

template <int IO>
static void dropout_t(const DropArgs& p, hipStream_t stream) {
    const dim3 block(256);
    const uintptr_t at = reinterpret_cast<uintptr_t>(p.x) | reinterpret_cast<uintptr_t>(p.residual) | reinterpret_cast<uintptr_t>(p.y);
    const bool vec = (at & 15) == 0;
    if (p.shared > 1 && p.inner % 8 == 0 && vec) {
        const long long blocks = (p.outer * (p.inner / 8) + 255) / 256;
        // about 4096 workgroups, at least four shared positions per draw of the mask
        const long long want = max(1LL, min((p.shared + 3) / 4, (4096 + blocks - 1) / blocks));
        const long long per = (p.shared + want - 1) / want;
        if ((p.shared + per - 1) / per <= 65535 && per <= 0x7fffffff) {
            hipLaunchKernelGGL((dropout_shared_kernel<IO, 4>), dim3((unsigned)blocks, (unsigned)((p.shared + per - 1) / per)),
                               block, 0, stream, p, (int)per);
            return;
        }
    }
    const dim3 grid((unsigned)(((p.outer * p.shared * p.inner + 7) / 8 + 255) / 256));
    if (p.shared == 1) {
        if (vec) hipLaunchKernelGGL((dropout_flat_kernel<IO, true, false>), grid, block, 0, stream, p);
        else hipLaunchKernelGGL((dropout_flat_kernel<IO, false, false>), grid, block, 0, stream, p);
    } else {
        if (vec) hipLaunchKernelGGL((dropout_flat_kernel<IO, true, true>), grid, block, 0, stream, p);
        else hipLaunchKernelGGL((dropout_flat_kernel<IO, false, true>), grid, block, 0, stream, p);
    }
}

void launch_dropout(const DropArgs& p, int io_dtype, hipStream_t stream) {
    if (io_dtype == KFH_F32) dropout_t<KFH_F32>(p, stream);
    else dropout_t<KFH_BF16>(p, stream);
}

}  // namespace kfh
