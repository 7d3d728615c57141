// Gated feed-forward block in bf16 for many rows of C = 64, 128 or 256 channels (the pair track's
// widths); the formulas are in gatedffn.hip.
#include "ffn_tiles.hpp"

namespace kfh {

// ---------------------------------------------------------------------------------------------
// Many rows of C = 64, 128 or 256 channels in bf16 (the pair track's widths): rows stay, weights
// stream.  A wavefront holds the MFMA fragments of 32 rows of x (and dy) in registers for the whole
// kernel; each step brings the weights of 32 hidden channels, packed as MFMA fragments, through
// double-buffered LDS and computes u, v (and dh) as D[hidden][row].  The rounded accumulators are by
// themselves the row operand of the next product (K_ACC order), so
//   forward,  FUSE: y += h W_out^T stays in registers, h never leaves them
//   backward, FUSE: dx += [du dv] W_in likewise; du, dv and h are written for the weight gradients
// FUSE needs C / 2 accumulator registers more, which C = 256 does not have; there the second product
// is a launch of its own.  Bound by three things of about the same length, of which the wavefronts of a SIMD
// overlap a part: the products, the LDS reads of the weights (one 1 KiB fragment per MFMA) and the activation's
// VALU work; the backward kernels also by the 6 F bytes a row that they write.  589824 x 128 x 256 forward 134 us
// (0.86 PF/s), 147456 x 128 x 256 backward with dx 92 us, 146689 x 256 x 1024 backward without dx 357 us.
// ---------------------------------------------------------------------------------------------
template <int KS, bool BWD, bool FUSE> constexpr int stream_frags() {
    return (BWD ? 3 : 2) * KS + (FUSE ? (BWD ? 2 : 1) * KS : 0);
}
// output channel of accumulator block n, column col: NI adjacent channels per lane
template <int KS> __host__ __device__ constexpr int stream_chan(int n, int col) {
    constexpr int NI = KS / 2 < 4 ? KS / 2 : 4;
    return (n / NI) * 32 * NI + NI * col + n % NI;
}

// Packed weights of a step of 32 hidden channels f0.., 1 KiB per fragment, lane-major:
//   KS x W_in rows f0.. (u), KS x W_in rows F + f0.. (v), [BWD] KS x W_out columns f0.. (dh),
//   [FUSE] forward: KS x W_out as B operand (block n, k-step); backward: KS x W_in u rows, KS x v rows
template <int KS, bool BWD, bool FUSE>
__global__ __launch_bounds__(256) void ffn_pack_kernel(const uint16_t* __restrict__ w_in, const uint16_t* __restrict__ w_out,
                                                       u32x4* __restrict__ dst, int F, long long slots) {
    constexpr int C = 16 * KS, NF = stream_frags<KS, BWD, FUSE>();
    const long long slot = (long long)blockIdx.x * 256 + threadIdx.x;
    if (slot >= slots) return;
    const int lane = (int)(slot & 63), fr = (int)((slot >> 6) % NF);
    const int f0 = (int)((slot >> 6) / NF) * 32, col = lane & 31, half = lane >> 5;
    const int group = fr / KS, ks = fr % KS;
    uint32_t v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const int c = 16 * ks + 8 * half + e;                           // contraction over channels
        const int f = f0 + 16 * (ks & 1) + 8 * (e >> 2) + 4 * half + (e & 3);    // over hidden (K_ACC)
        size_t src;
        const uint16_t* w = w_in;
        if (group < 2) src = (size_t)(group * F + f0 + col) * C + c;
        else if (BWD && group == 2) { w = w_out; src = (size_t)c * F + f0 + col; }
        else if (!BWD) { w = w_out; src = (size_t)stream_chan<KS>(ks >> 1, col) * F + f; }
        else src = (size_t)((group - 3) * F + f) * C + stream_chan<KS>(ks >> 1, col);
        v[e] = w[src];
    }
    dst[slot] = u32x4{v[0] | (v[1] << 16), v[2] | (v[3] << 16), v[4] | (v[5] << 16), v[6] | (v[7] << 16)};
}

// the two fragments of a block of 32 rows x 32 hidden channels, as they are: 1 KiB per store, past the
// caches, which hold the weights.  Hidden values of 146689 x 256 x 1024: without any stores 248 us; row by
// row in 32-byte pieces 462, whole fragments 408, past the caches 352.  Rows behind the last are zeros, for the sums over rows.
__device__ __forceinline__ void store_hidden(uint16_t* t, size_t slot, bool live, const bf16x8& f0, const bf16x8& f1) {
    const u32x4 none = {0u, 0u, 0u, 0u};
    u32x4* const o = reinterpret_cast<u32x4*>(t) + slot;
    __builtin_nontemporal_store(live ? __builtin_bit_cast(u32x4, f0) : none, o);
    __builtin_nontemporal_store(live ? __builtin_bit_cast(u32x4, f1) : none, o + 64);
}

template <int KS, bool BWD, bool FUSE, int NW>
__device__ __forceinline__ void stream_rows(const uint16_t* __restrict__ x, const uint16_t* __restrict__ dy,
                                            const u32x4* __restrict__ wp, uint16_t* __restrict__ h, uint16_t* __restrict__ d,
                                            uint16_t* __restrict__ out, long long M, int F) {
    constexpr int C = 16 * KS, NF = stream_frags<KS, BWD, FUSE>(), NT = NW * 64, NB = FUSE ? KS / 2 : 1;
    // backward: the weights of the next step come in two halves, one during the first products and one during
    // the activation and the second products, with half the registers on the way (147456 x 128 x 256: 179 ->
    // 162 us); forward: during the activation and the second products
    constexpr int SLOTS = NF * 64, NPRE = (SLOTS + NT - 1) / NT, H0 = BWD ? (NPRE + 1) / 2 : NPRE;
    __shared__ __attribute__((aligned(16))) u32x4 smem[2 * SLOTS];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, col = lane & 31, half = lane >> 5;
    const long long p0 = (long long)blockIdx.x * (32 * NW) + wave * 32;
    const int steps = F / 32;
    u32x4 pre[H0];
    auto fetch = [&](int s, auto part) {
        constexpr int I0 = decltype(part)::v ? H0 : 0, I1 = decltype(part)::v ? NPRE : H0;
#pragma unroll
        for (int i = I0; i < I1; ++i) pre[i - I0] = wp[(size_t)s * SLOTS + (SLOTS % NT ? min(i * NT + tid, SLOTS - 1) : i * NT + tid)];
    };
    auto commit = [&](int b, auto part) {
        constexpr int I0 = decltype(part)::v ? H0 : 0, I1 = decltype(part)::v ? NPRE : H0;
#pragma unroll
        for (int i = I0; i < I1; ++i)
            if (SLOTS % NT == 0 || i * NT + tid < SLOTS) smem[b * SLOTS + i * NT + tid] = pre[i - I0];
    };
    fetch(0, Int<0>{});
    const long long p = p0 + col;
    const bool live = p < M;
    const size_t row = (size_t)min(p, M - 1) * C + 8 * half;
    bf16x8 xf[KS], yf[BWD ? KS : 1];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) xf[ks] = *reinterpret_cast<const bf16x8*>(x + row + 16 * ks);
    if constexpr (BWD) {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) yf[ks] = *reinterpret_cast<const bf16x8*>(dy + row + 16 * ks);
    }
    commit(0, Int<0>{});
    fetch(0, Int<1>{});
    commit(0, Int<1>{});
    __syncthreads();
    f32x16 oacc[NB];
    if constexpr (FUSE) {
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int v = 0; v < 16; ++v) oacc[n][v] = 0.f;
    }
    f32x16 u, v, g;
    auto products = [&](const bf16x8* w) {
#pragma unroll
        for (int i = 0; i < 16; ++i) { u[i] = 0.f; v[i] = 0.f; g[i] = 0.f; }
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            u = mfma32(w[ks * 64], xf[ks], u);
            v = mfma32(w[(KS + ks) * 64], xf[ks], v);
            if constexpr (BWD) g = mfma32(w[(2 * KS + ks) * 64], yf[ks], g);
        }
    };
    // activation of step s, its second product (FUSE) and its stores
    auto finish = [&](int s, const bf16x8* w) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float sg = sigmoidf_fast(u[i]), us = u[i] * sg;
            if constexpr (BWD) {
                const float gg = g[i], vv = v[i];
                g[i] = us * vv;                                          // h
                u[i] = gg * vv * (sg + us * (1.f - sg));                 // du
                v[i] = gg * us;                                          // dv
            } else {
                u[i] = us * v[i];                                        // h
            }
        }
        bf16x8 a0, a1;
        acc_to_frags(u, a0, a1);
        if constexpr (BWD) {
            bf16x8 b0, b1, h0, h1;
            acc_to_frags(v, b0, b1);
            acc_to_frags(g, h0, h1);
            if constexpr (FUSE) {
#pragma unroll
                for (int n = 0; n < NB; ++n) {
                    oacc[n] = mfma32(a0, w[(3 * KS + 2 * n) * 64], oacc[n]);
                    oacc[n] = mfma32(a1, w[(3 * KS + 2 * n + 1) * 64], oacc[n]);
                    oacc[n] = mfma32(b0, w[(4 * KS + 2 * n) * 64], oacc[n]);
                    oacc[n] = mfma32(b1, w[(4 * KS + 2 * n + 1) * 64], oacc[n]);
                }
            }
            if (p0 < M) {
                store_hidden(h, hidden_slot(p, s, F / 32, 0, half), live, h0, h1);
                store_hidden(d, hidden_slot(p, s, F / 16, 0, half), live, a0, a1);
                store_hidden(d, hidden_slot(p, F / 32 + s, F / 16, 0, half), live, b0, b1);
            }
        } else if constexpr (FUSE) {
#pragma unroll
            for (int n = 0; n < NB; ++n) {
                oacc[n] = mfma32(a0, w[(2 * KS + 2 * n) * 64], oacc[n]);
                oacc[n] = mfma32(a1, w[(2 * KS + 2 * n + 1) * 64], oacc[n]);
            }
        } else {
            if (p0 < M) store_hidden(h, hidden_slot(p, s, F / 32, 0, half), live, a0, a1);
        }
    };
    for (int s = 0; s < steps; ++s) {
        if (BWD && s + 1 < steps) fetch(s + 1, Int<0>{});
        const bf16x8* w = reinterpret_cast<const bf16x8*>(smem + (s & 1) * SLOTS) + lane;
        __builtin_amdgcn_s_setprio(1);        // before the wavefronts that are in their activations: 1-3 %
        products(w);
        __builtin_amdgcn_s_setprio(0);
        if (s + 1 < steps) {
            if constexpr (BWD) {
                commit((s + 1) & 1, Int<0>{});
                fetch(s + 1, Int<1>{});
            } else {
                fetch(s + 1, Int<0>{});
            }
        }
        finish(s, w);
        if (s + 1 < steps) commit((s + 1) & 1, Int<(BWD ? 1 : 0)>{});
        __syncthreads();
    }
    if constexpr (FUSE) {
        if (!out) return;                                                // no dx asked for
        constexpr int NI = NB < 4 ? NB : 4;
#pragma unroll
        for (int v = 0; v < 16; ++v) {
            const long long q = p0 + acc_row(v, half);
            if (q >= M) continue;
#pragma unroll
            for (int n = 0; n < NB; n += NI) {
                uint16_t* o = out + (size_t)q * C + stream_chan<KS>(n, col);
                if constexpr (NI == 4)
                    *reinterpret_cast<u32x2*>(o) = u32x2{pack_bf16(oacc[n][v], oacc[n + 1][v]), pack_bf16(oacc[n + 2][v], oacc[n + 3][v])};
                else
                    *reinterpret_cast<uint32_t*>(o) = pack_bf16(oacc[n][v], oacc[n + 1][v]);
            }
        }
    }
}

// a name per workgroup size: up to C = 128 workgroups of 4 wavefronts (backward two, forward three on a CU), at
// C = 256 one of 8
template <int KS, bool BWD>
__global__ __launch_bounds__(256, (BWD ? 2 : 3)) void ffn_stream_kernel(const uint16_t* __restrict__ x, const uint16_t* __restrict__ dy,
                                                                        const u32x4* __restrict__ wp, uint16_t* __restrict__ h,
                                                                        uint16_t* __restrict__ d, uint16_t* __restrict__ out,
                                                                        long long M, int F) {
    stream_rows<KS, BWD, true, 4>(x, dy, wp, h, d, out, M, F);
}
template <int KS, bool BWD>
__global__ __launch_bounds__(512, 2) void ffn_stream_wide_kernel(const uint16_t* __restrict__ x, const uint16_t* __restrict__ dy,
                                                                 const u32x4* __restrict__ wp, uint16_t* __restrict__ h,
                                                                 uint16_t* __restrict__ d, uint16_t* __restrict__ out,
                                                                 long long M, int F) {
    stream_rows<KS, BWD, false, 8>(x, dy, wp, h, d, out, M, F);
}

template <int KS, bool BWD>
static void stream_t(const void* x, const void* dy, const void* w_in, const void* w_out, void* pack, void* h, void* d,
                     void* out, long long M, int F, hipStream_t stream) {
    constexpr bool FUSE = KS <= 8;
    constexpr int NW = FUSE ? 4 : 8;
    const long long slots = (long long)(F / 32) * stream_frags<KS, BWD, FUSE>() * 64;
    hipLaunchKernelGGL((ffn_pack_kernel<KS, BWD, FUSE>), dim3((unsigned)((slots + 255) / 256)), dim3(256), 0, stream,
                       static_cast<const uint16_t*>(w_in), static_cast<const uint16_t*>(w_out), static_cast<u32x4*>(pack), F,
                       slots);
    const dim3 grid((unsigned)((M + 32 * NW - 1) / (32 * NW))), block(NW * 64);
    const uint16_t* const xs = static_cast<const uint16_t*>(x);
    const uint16_t* const dys = static_cast<const uint16_t*>(dy);
    const u32x4* const wp = static_cast<const u32x4*>(pack);
    uint16_t* const hs = static_cast<uint16_t*>(h);
    uint16_t* const ds = static_cast<uint16_t*>(d);
    uint16_t* const outs = static_cast<uint16_t*>(out);
    if constexpr (FUSE)
        hipLaunchKernelGGL((ffn_stream_kernel<KS, BWD>), grid, block, 0, stream, xs, dys, wp, hs, ds, outs, M, F);
    else
        hipLaunchKernelGGL((ffn_stream_wide_kernel<KS, BWD>), grid, block, 0, stream, xs, dys, wp, hs, ds, outs, M, F);
}

size_t ffn_stream_pack_bytes(int C, int F, int backward) {
    const int KS = C / 16, nf = (backward ? 3 : 2) * KS + (C <= 128 ? (backward ? 2 : 1) * KS : 0);
    return (size_t)(F / 32) * nf * 1024;
}

void launch_ffn_stream(const void* x, const void* dy, const void* w_in, const void* w_out, void* pack, void* h, void* d,
                       void* out, long long M, int C, int F, hipStream_t stream) {
    if (dy) {
        if (C == 64) stream_t<4, true>(x, dy, w_in, w_out, pack, h, d, out, M, F, stream);
        else if (C == 128) stream_t<8, true>(x, dy, w_in, w_out, pack, h, d, out, M, F, stream);
        else stream_t<16, true>(x, dy, w_in, w_out, pack, h, d, out, M, F, stream);
    } else {
        if (C == 64) stream_t<4, false>(x, dy, w_in, w_out, pack, h, d, out, M, F, stream);
        else if (C == 128) stream_t<8, false>(x, dy, w_in, w_out, pack, h, d, out, M, F, stream);
        else stream_t<16, false>(x, dy, w_in, w_out, pack, h, d, out, M, F, stream);
    }
}

}  // namespace kfh
