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
// from memory to registers (fetch) to LDS (commit), where it is stored [part][row][BK + 8] bf16, so
// that the 8 k-consecutive values of an MFMA fragment are one 16-byte read; the 8 values of padding
// keep consecutive rows on different banks.
//   K_MAJOR : memory is [row][k], k contiguous: a thread moves 8 k of a row
//   R_MAJOR : memory is [k][row], rows contiguous: a thread loads 4 k x 8 rows and writes them
//             transposed, 4 k (8 bytes) per row
//   K_BLOCK, R_BLOCK: the same two for hidden values written by ffn_stream_kernel, blocks of 32 rows x
//             32 channels (ld: channels) of two MFMA fragments each: hidden_slot
// Values outside [row < rmax, k < kmax] are zeros: their addresses are kept inside the tensor, so that
// no load sits behind a branch, and the values cleared when they are committed.
// ---------------------------------------------------------------------------------------------
template <int IO> constexpr int parts_of() { return IO == KFH_F32 ? 3 : 1; }

template <int IO> struct Raw8;                               // 8 values as they come from memory
template <> struct Raw8<KFH_BF16> {
    u32x4 w;
    __device__ __forceinline__ void get(const char* p, uint32_t o) { w = *reinterpret_cast<const u32x4*>(p + o); }
    __device__ __forceinline__ void clear() { w = u32x4{0u, 0u, 0u, 0u}; }
};
template <> struct Raw8<KFH_F32> {
    f32x4 a, b;
    __device__ __forceinline__ void get(const char* p, uint32_t o) {
        const f32x4* s = reinterpret_cast<const f32x4*>(p + o);
        a = s[0];
        b = s[1];
    }
    __device__ __forceinline__ void clear() { a = b = f32x4{0.f, 0.f, 0.f, 0.f}; }
    __device__ __forceinline__ float at(int i) const { return i < 4 ? a[i & 3] : b[i & 3]; }
};

enum : int { K_MAJOR = 0, R_MAJOR, K_BLOCK, R_BLOCK };

// 16-byte slot of the 8 channels 16 ks + 4 half + {0..3, 8..11} of block (m / 32, channel block hb), row m
__device__ __forceinline__ size_t hidden_slot(long long m, int hb, int nhb, int ks, int half) {
    return ((size_t)((m >> 5) * nhb + hb) * 2 + ks) * 64 + half * 32 + (m & 31);
}

template <int IO, int KIND, int ROWS, int BK, int NT = 256>
struct TileLoad {
    static constexpr bool KC = KIND == K_MAJOR || KIND == K_BLOCK;
    static constexpr int PARTS = parts_of<IO>();
    static constexpr int LDK = BK + 8;                       // bf16 per stored row
    static constexpr int PLANE = ROWS * LDK;                 // bf16 per part
    static constexpr int UNITS = KC ? ROWS * BK / 8 : ROWS * BK / 32;
    static constexpr int NU = (UNITS + NT - 1) / NT;           // units per thread
    static constexpr int NV = KC ? 1 : 4;                    // 8-value vectors per unit
    static constexpr int ES = IO == KFH_F32 ? 4 : 2;
    Raw8<IO> v[NU][NV];
    const char* base;                                        // of the tile's first row; the same in all lanes
    long long step, vec;                                     // bytes from a k to the next, from a vector of a unit to the next
    uint32_t off[NU];                                        // bytes from base of unit i at k = 0
    unsigned off_rows, bad;                                  // bit i * NV + j: vector j of unit i lies outside (rows only / in all)

    // k of unit u inside the tile
    static __device__ __forceinline__ int unit_k(int u) {
        return KIND == K_MAJOR ? (u % (BK / 8)) * 8 : KIND == K_BLOCK ? (u / ROWS) * 8 : (u % (BK / 4)) * 4;
    }
    // what does not change along the contraction: every later address is base + k * step + off + j * vec.
    // A row behind the last reads the last one's values, which commit clears.
    __device__ __forceinline__ void init(const void* src, long long ld, long long row0, long long rmax, int tid) {
        const int left = (int)min(rmax - row0, (long long)ROWS);          // rows of this tile
        const int nhb = (int)(ld >> 5);
        off_rows = 0;
        const char* const s = static_cast<const char*>(src);
        if constexpr (KIND == K_MAJOR) { base = s + row0 * ld * ES; step = ES; vec = 0; }
        else if constexpr (KIND == R_MAJOR) { base = s + row0 * ES; step = vec = ld * ES; }
        else if constexpr (KIND == K_BLOCK) { base = s + (row0 >> 5) * nhb * 2048; step = 64; vec = 0; }   // 32 k: 2 KiB
        else { base = s + (row0 >> 5) * 2048; step = (long long)nhb * 64; vec = 16; }                       // 32 k: nhb blocks
#pragma unroll
        for (int i = 0; i < NU; ++i) {
            const int u = min(i * NT + tid, UNITS - 1), k = unit_k(u);
            int r = KIND == K_MAJOR ? u / (BK / 8) : KIND == K_BLOCK ? u % ROWS : (u / (BK / 4)) * 8;
            if (r >= left) {
                off_rows |= ((1u << NV) - 1) << (i * NV);
                r = KC ? left - 1 : left - 8;
            }
            if constexpr (KIND == K_MAJOR) off[i] = (uint32_t)(r * (int)ld + k) * ES;
            else if constexpr (KIND == R_MAJOR) off[i] = (uint32_t)(k * (int)ld + r) * ES;
            else if constexpr (KIND == K_BLOCK)
                off[i] = (uint32_t)(((r >> 5) * nhb + (k >> 5)) * 128 + ((k >> 3) & 3) * 32 + (r & 31)) * 16;
            else
                off[i] = (uint32_t)(((k >> 5) * nhb + (r >> 5)) * 128 + ((r >> 3) & 3) * 32 + (k & 31)) * 16;
        }
    }
    // the tile at k0 < kmax; only a tile that reaches behind kmax looks at single vectors (they read the
    // tile's first k instead, which lies inside)
    __device__ __forceinline__ void fetch(long long k0, long long kmax, int tid) {
        const char* const b = base + k0 * step;
        bad = off_rows;
        if (k0 + BK <= kmax) {
#pragma unroll
            for (int i = 0; i < NU; ++i)
#pragma unroll
                for (int j = 0; j < NV; ++j) v[i][j].get(b + j * vec, off[i]);
        } else {
#pragma unroll
            for (int i = 0; i < NU; ++i) {
                const int k = unit_k(min(i * NT + tid, UNITS - 1));
                // off of the same row at k = 0
                uint32_t first = off[i];
                if constexpr (KIND == K_MAJOR || KIND == R_MAJOR) first -= (uint32_t)(k * step);
                else if constexpr (KIND == K_BLOCK) first -= (uint32_t)((k >> 5) * 128 + ((k >> 3) & 3) * 32) * 16;
                else first -= (uint32_t)((k >> 5) * 32 * step) + (k & 31) * 16;
#pragma unroll
                for (int j = 0; j < NV; ++j) {
                    const bool out = k0 + k + j >= kmax;
                    bad |= (unsigned)out << (i * NV + j);
                    v[i][j].get(out ? b : b + j * vec, out ? first : off[i]);
                }
            }
        }
    }
    __device__ __forceinline__ void commit(uint16_t* lds, int tid) {
        if (bad) {
#pragma unroll
            for (int i = 0; i < NU; ++i)
#pragma unroll
                for (int j = 0; j < NV; ++j)
                    if ((bad >> (i * NV + j)) & 1) v[i][j].clear();
        }
#pragma unroll
        for (int i = 0; i < NU; ++i) {
            const int u = i * NT + tid;
            if (UNITS % NT != 0 && u >= UNITS) continue;
            if constexpr (KIND == K_BLOCK) {
                const int g = u / ROWS;                      // group 4 b + 2 ks + half: channels 32 b + 16 ks + 4 half + {0..3, 8..11}
                uint16_t* d = lds + (u % ROWS) * LDK + (g >> 1) * 16 + (g & 1) * 4;
                *reinterpret_cast<u32x2*>(d) = u32x2{v[i][0].w[0], v[i][0].w[1]};
                *reinterpret_cast<u32x2*>(d + 8) = u32x2{v[i][0].w[2], v[i][0].w[3]};
            } else if constexpr (KC) {
                uint16_t* d = lds + (u / (BK / 8)) * LDK + (u % (BK / 8)) * 8;
                if constexpr (PARTS == 1) {
                    *reinterpret_cast<u32x4*>(d) = v[i][0].w;
                } else {
                    float q[8][3];
#pragma unroll
                    for (int e = 0; e < 8; ++e) split3(v[i][0].at(e), q[e]);
#pragma unroll
                    for (int p = 0; p < 3; ++p) {
                        u32x4 w;
#pragma unroll
                        for (int e = 0; e < 4; ++e) w[e] = pack_bf16(q[2 * e][p], q[2 * e + 1][p]);
                        *reinterpret_cast<u32x4*>(d + p * PLANE) = w;
                    }
                }
            } else {
                const int g = u / (BK / 4);
                uint16_t* const d0 = lds + (KIND == R_BLOCK ? (g >> 1) * 16 + (g & 1) * 4 : g * 8) * LDK + (u % (BK / 4)) * 4;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    uint16_t* const d = d0 + (KIND == R_BLOCK ? 8 * (e >> 2) + (e & 3) : e) * LDK;
                    if constexpr (PARTS == 1) {
                        // half-word e of the four vectors
                        const uint32_t a = v[i][0].w[e >> 1], b = v[i][1].w[e >> 1], c = v[i][2].w[e >> 1], f = v[i][3].w[e >> 1];
                        const u32x2 w = (e & 1) ? u32x2{(a >> 16) | (b & 0xffff0000u), (c >> 16) | (f & 0xffff0000u)}
                                                : u32x2{(a & 0xffffu) | (b << 16), (c & 0xffffu) | (f << 16)};
                        *reinterpret_cast<u32x2*>(d) = w;
                    } else {
                        float q[4][3];
#pragma unroll
                        for (int j = 0; j < 4; ++j) split3(v[i][j].at(e), q[j]);
#pragma unroll
                        for (int p = 0; p < 3; ++p) {
                            u32x2 w = {pack_bf16(q[0][p], q[1][p]), pack_bf16(q[2][p], q[3][p])};
                            *reinterpret_cast<u32x2*>(d + p * PLANE) = w;
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

// Workgroups are dealt to the 8 XCDs in turn, each with an L2 of its own: the `nt` tiles that share a
// row tile follow each other on one XCD, so its rows are read from memory once (without it the weight
// gradient 2048 x 256 over 146689 rows took 287 us instead of 198).  With few row tiles, unless they
// divide evenly, that would leave XCDs idle, and the tiles are simply counted through.
__host__ __device__ constexpr bool xcd_dealt(long long mtiles) { return mtiles >= 64 || mtiles % 8 == 0; }
__device__ __forceinline__ bool xcd_tile(long long id, long long mtiles, int nt, long long& mt, int& n) {
    const bool dealt = xcd_dealt(mtiles);
    const long long slot = dealt ? id >> 3 : id;
    mt = slot / nt;
    n = (int)(slot - mt * nt);
    if (dealt) mt = mt * 8 + (id & 7);
    return mt < mtiles;
}
static unsigned xcd_grid(long long mtiles, int nt) {
    return (unsigned)((xcd_dealt(mtiles) ? (mtiles + 7) / 8 * 8 : mtiles) * nt);
}

// A finished tile of RM rows x RN columns goes through LDS so that it leaves in whole rows (16 bytes a
// lane, 2 RN bytes a row) instead of 8 bytes of 64 different rows.  put: four consecutive columns.
template <int IO, int RM, int RN, int NT = 256>
struct TileStore {
    static constexpr int ES = IO == KFH_F32 ? 4 : 2;
    static constexpr int LD = RN * ES + 16;                  // bytes per staged row
    static constexpr int BYTES = RM * LD;
    static __device__ __forceinline__ void put(char* t, int r, int c, float a, float b, float d, float e) {
        store4<IO>(t + r * LD, (size_t)c, a, b, d, e);
    }
    static __device__ __forceinline__ void flush(const char* t, void* out, long long ld, long long m0, long long M, int n0,
                                                 int N, int tid) {
        constexpr int PER = RN * ES / 16;                    // 16-byte pieces per row
#pragma unroll
        for (int i = 0; i < RM * PER / NT; ++i) {
            const int u = i * NT + tid, r = u / PER, c = (u % PER) * (16 / ES);
            if (m0 + r < M && n0 + c < N)
                *reinterpret_cast<u32x4*>(static_cast<char*>(out) + ((size_t)(m0 + r) * ld + n0 + c) * ES) =
                    *reinterpret_cast<const u32x4*>(t + r * LD + c * ES);
        }
    }
};

// ---------------------------------------------------------------------------------------------
// Hidden values of a tile of TM rows x 64 hidden channels; wavefront (wm, wn) owns TM / 2 rows x 32
// channels of u and v (and dh: the same accumulator shape, from dy and w_out).
//   forward : h [M, F]
//   backward: d [M, 2F] = (du, dv) and h [M, F]
// The next k-tile travels from memory while the matrix cores work on the present one.
// ---------------------------------------------------------------------------------------------
template <int IO, int TM> constexpr int hidden_lds(bool bwd) {
    constexpr int BK = IO == KFH_F32 ? 32 : 64;
    const int in = parts_of<IO>() * (TM + 128) * (BK + 8) * 2;
    const int out = (bwd ? 3 : 1) * TileStore<IO, TM, 64>::BYTES;
    return in > out ? in : out;
}

template <int IO, bool BWD, int TM>
__global__ __launch_bounds__(256) void ffn_hidden_kernel(const void* __restrict__ x, const void* __restrict__ dy,
                                                         const void* __restrict__ w_in,
                                                         const void* __restrict__ w_out, void* __restrict__ h,
                                                         void* __restrict__ d, long long M, int C, int F) {
    constexpr int BK = IO == KFH_F32 ? 32 : 64, LDK = BK + 8, P = parts_of<IO>(), NA = TM / 64;
    __shared__ __attribute__((aligned(16))) char smem[hidden_lds<IO, TM>(BWD)];
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
    TileLoad<IO, K_MAJOR, TM, BK> lx;
    TileLoad<IO, K_MAJOR, 64, BK> lu, lv;
    TileLoad<IO, R_MAJOR, 64, BK> lo;
    lx.init(x, C, m0, M, tid);
    lu.init(w_in, C, f0, F, tid);
    lv.init(w_in, C, (long long)F + f0, 2LL * F, tid);
    lx.fetch(0, C, tid); lu.fetch(0, C, tid); lv.fetch(0, C, tid);
    for (int k0 = 0; k0 < C; k0 += BK) {
        __syncthreads();
        lx.commit(sa, tid); lu.commit(su, tid); lv.commit(sv, tid);
        __syncthreads();
        if (k0 + BK < C) {
            lx.fetch(k0 + BK, C, tid); lu.fetch(k0 + BK, C, tid); lv.fetch(k0 + BK, C, tid);
        } else if (BWD) {
            lx.init(dy, C, m0, M, tid);
            lo.init(w_out, F, f0, F, tid);
            lx.fetch(0, C, tid); lo.fetch(0, C, tid);
        }
        tile_mma<IO, NA, 1, TM, 64, BK>(sa, wm * (TM / 2), su, wn * 32, lane, u);
        tile_mma<IO, NA, 1, TM, 64, BK>(sa, wm * (TM / 2), sv, wn * 32, lane, v);
    }
    if constexpr (BWD) {
        for (int k0 = 0; k0 < C; k0 += BK) {
            __syncthreads();
            lx.commit(sa, tid); lo.commit(su, tid);
            __syncthreads();
            if (k0 + BK < C) {
                lx.fetch(k0 + BK, C, tid); lo.fetch(k0 + BK, C, tid);
            }
            tile_mma<IO, NA, 1, TM, 64, BK>(sa, wm * (TM / 2), su, wn * 32, lane, g);
        }
    }
    __syncthreads();
    using Out = TileStore<IO, TM, 64>;
    char* const th = smem;
    char* const tu = smem + Out::BYTES;
    char* const tv = smem + 2 * Out::BYTES;
#pragma unroll
    for (int a = 0; a < NA; ++a) {
        const int r = wm * (TM / 2) + 32 * a + (lane & 31);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int f = wn * 32 + 8 * q + 4 * (lane >> 5);
            float hh[4], du[4], dv[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float uu = u[a][0][4 * q + e], vv = v[a][0][4 * q + e];
                const float s = sigmoidf_fast(uu), us = uu * s;
                hh[e] = us * vv;
                if constexpr (BWD) {
                    const float gg = g[a][0][4 * q + e];
                    dv[e] = gg * us;
                    du[e] = gg * vv * (s + us * (1.f - s));
                }
            }
            Out::put(th, r, f, hh[0], hh[1], hh[2], hh[3]);
            if constexpr (BWD) {
                Out::put(tu, r, f, du[0], du[1], du[2], du[3]);
                Out::put(tv, r, f, dv[0], dv[1], dv[2], dv[3]);
            }
        }
    }
    __syncthreads();
    Out::flush(th, h, F, m0, M, f0, F, tid);
    if constexpr (BWD) {
        Out::flush(tu, d, 2LL * F, m0, M, f0, F, tid);
        Out::flush(tv, static_cast<char*>(d) + (size_t)F * Out::ES, 2LL * F, m0, M, f0, F, tid);
    }
}

// ---------------------------------------------------------------------------------------------
// out[m][n] = sum_k A(m, k) B(n, k); AK / BK_ as TileLoad's KIND; a workgroup of NW wavefronts owns
// TM x TN results, wavefront (wm, wn) TM / WM x TN / WN of them.  The contraction is cut into `splits`
// ranges of kper; with more than one the results are fp32 partial tiles at out + range * Mo * No (PART),
// else they are written as IO.
//
// What bounds it is the way of the operands into LDS: with 128 x 128 tiles the weight gradient 2048 x 256
// over 146689 rows takes 261 us for the loads alone, 100 us for the products alone (1.5 PF/s) and 265 us
// together.  A 256 x 256 tile asks for half the bytes.
// ---------------------------------------------------------------------------------------------
template <int V> struct Int { static constexpr int v = V; };
template <int TM, int TN> struct Waves {                     // wavefronts of a tile and their arrangement
    static constexpr int NW = TM * TN >= 256 * 128 ? 8 : 4;
    static constexpr int WM = NW == 4 || TM < TN || TM == TN ? 2 : 4, WN = NW / WM;
};
template <int IO, int TM, int TN, bool PART> struct GemmLds {
    static constexpr int BK = IO == KFH_F32 ? 32 : 64, NT = Waves<TM, TN>::NW * 64;
    using Out = TileStore<PART ? (int)KFH_F32 : IO, TM, TN / Waves<TM, TN>::WN, NT>;      // one column of wavefronts
    static constexpr int IN = 2 * parts_of<IO>() * (TM + TN) * (BK + 8) * 2;
    static constexpr int BYTES = IN > Out::BYTES ? IN : Out::BYTES;
};

template <int IO, int AK, int BK_, bool PART, int TM, int TN>
__global__ __launch_bounds__((Waves<TM, TN>::NW * 64)) void ffn_gemm_kernel(
    const void* __restrict__ A, long long lda, const void* __restrict__ B, long long ldb, void* __restrict__ out,
    long long Mo, int No, long long K, long long kper, int splits) {
    using W = Waves<TM, TN>;
    using Lds = GemmLds<IO, TM, TN, PART>;
    constexpr int BK = Lds::BK, LDK = BK + 8, P = parts_of<IO>(), NT = Lds::NT;
    constexpr int RM = TM / W::WM, RN = TN / W::WN, NA = RM / 32, NB = RN / 32;
    __shared__ __attribute__((aligned(16))) char smem[Lds::BYTES];
    constexpr int BUF = P * (TM + TN) * LDK;
    uint16_t* const buf = reinterpret_cast<uint16_t*>(smem);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int wm = wave % W::WM, wn = wave / W::WM;
    const long long mtiles = (Mo + TM - 1) / TM;
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
    const long long m0 = mt * TM;
    const int n0 = nt * TN;
    const long long kb = z * kper, ke = min(kb + kper, K);
    f32x16 acc[NA][NB];
    zero_acc(acc);
    TileLoad<IO, AK, TM, BK, NT> la;
    TileLoad<IO, BK_, TN, BK, NT> lb;
    // two k-tiles ahead: while the matrix cores work on one from LDS, the next is written to the other LDS
    // buffer and the one after travels from memory to registers; one barrier per k-tile
    const long long steps = kb < ke ? (ke - kb + BK - 1) / BK : 0;
    auto fetch = [&](long long s) {
        if (s >= steps) return;
        la.fetch(kb + s * BK, ke, tid);
        lb.fetch(kb + s * BK, ke, tid);
    };
    la.init(A, lda, m0, Mo, tid);
    lb.init(B, ldb, n0, No, tid);
    auto commit = [&](long long s) {
        if (s >= steps) return;
        uint16_t* const b = buf + (s & 1) * BUF;
        la.commit(b, tid);
        lb.commit(b + P * TM * LDK, tid);
    };
    fetch(0);
    commit(0);
    fetch(1);
    __syncthreads();
    for (long long s = 0; s < steps; ++s) {
        commit(s + 1);
        fetch(s + 2);
        const uint16_t* const b = buf + (s & 1) * BUF;
        tile_mma<IO, NA, NB, TM, TN, BK>(b, wm * RM, b + P * TM * LDK, wn * RN, lane, acc);
        __syncthreads();
    }
    // through LDS, one column of wavefronts at a time
    using Out = typename Lds::Out;
    char* const base = static_cast<char*>(out) + (PART ? (size_t)z * Mo * No * 4 : 0);
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

// out[i] = sum of `parts` fp32 values part[z * n + i]: 64 lanes x 4 values per workgroup, its four
// wavefronts take every fourth part; a fixed order
__global__ __launch_bounds__(256) void ffn_sum_parts_kernel(const float* __restrict__ part, int parts, long long n,
                                                            void* __restrict__ out, int out_dtype) {
    __shared__ f32x4 red[4][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long long i = ((long long)blockIdx.x * 64 + lane) * 4;
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
    if (i < n) {
#pragma unroll 4
        for (int z = wave; z < parts; z += 4) {
            const f32x4 w = *reinterpret_cast<const f32x4*>(part + (size_t)z * n + i);
#pragma unroll
            for (int e = 0; e < 4; ++e) s[e] += w[e];
        }
    }
    red[wave][lane] = s;
    __syncthreads();
    if (wave != 0 || i >= n) return;
    float o[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = (red[0][lane][e] + red[1][lane][e]) + (red[2][lane][e] + red[3][lane][e]);
    if (out_dtype == KFH_BF16) store4<KFH_BF16>(out, (size_t)i, o[0], o[1], o[2], o[3]);
    else store4<KFH_F32>(out, (size_t)i, o[0], o[1], o[2], o[3]);
}

// ---------------------------------------------------------------------------------------------
// Many rows of C = 64, 128 or 256 channels in bf16 (the pair track's widths): rows stay, weights
// stream.  A wavefront holds the MFMA fragments of 32 rows of x (and dy) in registers for the whole
// kernel; each step brings the weights of 32 hidden channels, packed as MFMA fragments, through
// double-buffered LDS and computes u, v (and dh) as D[hidden][row].  The rounded accumulators are by
// themselves the row operand of the next product (K_ACC order), so
//   forward,  FUSE: y += h W_out^T stays in registers, h never leaves them
//   backward, FUSE: dx += [du dv] W_in likewise; du, dv and h are written for the weight gradients
// FUSE needs C / 2 accumulator registers more, which C = 256 does not have; there the second product
// is a launch of its own.  Bound by the LDS reads of the weights (one 1 KiB fragment per MFMA) and the
// activation's VALU work.
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

template <int KS, bool BWD, bool FUSE, int NW, int OCC>
__global__ __launch_bounds__(NW * 64, OCC) void ffn_stream_kernel(const uint16_t* __restrict__ x,
                                                                  const uint16_t* __restrict__ dy,
                                                                  const u32x4* __restrict__ wp, uint16_t* __restrict__ h,
                                                                  uint16_t* __restrict__ d, uint16_t* __restrict__ out, long long M,
                                                                  int F) {
    constexpr int C = 16 * KS, NF = stream_frags<KS, BWD, FUSE>(), NT = NW * 64, NB = FUSE ? KS / 2 : 1;
    constexpr int SLOTS = NF * 64, NPRE = (SLOTS + NT - 1) / NT;
    __shared__ __attribute__((aligned(16))) u32x4 smem[2 * SLOTS];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, col = lane & 31, half = lane >> 5;
    const long long p0 = (long long)blockIdx.x * (32 * NW) + wave * 32;
    const int steps = F / 32;
    u32x4 pre[NPRE];
    auto fetch = [&](int s) {
#pragma unroll
        for (int i = 0; i < NPRE; ++i) pre[i] = wp[(size_t)s * SLOTS + min(i * NT + tid, SLOTS - 1)];
    };
    auto commit = [&](int b) {
#pragma unroll
        for (int i = 0; i < NPRE; ++i)
            if (SLOTS % NT == 0 || i * NT + tid < SLOTS) smem[b * SLOTS + i * NT + tid] = pre[i];
    };
    fetch(0);
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
    commit(0);
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
        if (s + 1 < steps) fetch(s + 1);
        const bf16x8* w = reinterpret_cast<const bf16x8*>(smem + (s & 1) * SLOTS) + lane;
        products(w);
        finish(s, w);
        if (s + 1 < steps) commit((s + 1) & 1);
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

// Ranges of rows the weight gradients are summed over in parallel: one workgroup per CU with large tiles (as
// many as fit; more would only add partial sums), two with 64 x 64, at least 256 rows each.
struct Wgrad { Tile t; int splits; long long per; };
static Wgrad wgrad_plan(long long M, long long a, long long b, int io_dtype) {
    Wgrad w;
    const long long most = max(1LL, up_div(M, 256));
    w.t = pick_tile(a, b, most, io_dtype);
    const long long tiles = up_div(a, w.t.m) * up_div(b, w.t.n);
    w.splits = (int)min(min(max(1LL, (w.t.m * w.t.n > 128 * 128 ? 256 : 512) / tiles), most), 256LL);
    if (w.splits > 8) w.splits = w.splits / 8 * 8;           // whole rounds over the XCDs
    w.per = up_div(up_div(M, w.splits), 64) * 64;
    return w;
}
static size_t wgrad_part_bytes(long long M, int C, int F, int io_dtype) {
    const size_t a = (size_t)wgrad_plan(M, 2LL * F, C, io_dtype).splits * 2 * F * C * 4;
    const size_t b = (size_t)wgrad_plan(M, C, F, io_dtype).splits * F * C * 4;
    return a > b ? a : b;
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

// The streamed kernels: bf16, a width they are built for, whole steps of hidden channels, and rows enough
// to give every CU a workgroup (below that their 128 or 256 rows per workgroup leave CUs idle).
static bool streamed(long long M, int C, int F, int io_dtype) {
    return io_dtype == KFH_BF16 && (C == 64 || C == 128 || C == 256) && F % 32 == 0 && M >= 16384;
}
static size_t stream_pack_bytes(int C, int F, int backward) {
    const int KS = C / 16, nf = (backward ? 3 : 2) * KS + (C <= 128 ? (backward ? 2 : 1) * KS : 0);
    return (size_t)(F / 32) * nf * 1024;
}

// workspace: h [M, F] (not in a fused forward call), backward: d [M, 2F], row-major or (streamed) in
// blocks; packed weights of the
// streamed kernels; partial sums
struct FfnWs { size_t h, d, pack, part, total; };
static FfnWs ffn_ws(long long M, int C, int F, int backward, int io_dtype) {
    const size_t e = io_dtype == KFH_F32 ? 4 : 2;
    const bool st = streamed(M, C, F, io_dtype), fused = st && C <= 128;
    const size_t rows = st ? (size_t)up_div(M, 32) * 32 : (size_t)M;         // whole blocks
    FfnWs w;
    w.h = 0;
    w.d = w.h + (backward || !fused ? up256(rows * F * e) : 0);
    w.pack = w.d + (backward ? up256(rows * 2 * F * e) : 0);
    w.part = w.pack + (st ? up256(stream_pack_bytes(C, F, backward)) : 0);
    size_t part = fused ? 0 : product_part_bytes(M, C, backward ? 2LL * F : F, io_dtype);
    if (backward) part = max(part, wgrad_part_bytes(M, C, F, io_dtype));
    w.total = w.part + up256(part);
    return w;
}
size_t gated_ffn_ws_bytes(long long M, int C, int F, int backward, int io_dtype) {
    return ffn_ws(M, C, F, backward, io_dtype).total;
}

static void sum_parts(const float* part, int parts, long long n, void* out, int out_dtype, hipStream_t stream) {
    hipLaunchKernelGGL(ffn_sum_parts_kernel, dim3((unsigned)up_div(n, 256)), dim3(256), 0, stream, part, parts, n, out,
                       out_dtype);
}

template <int IO, bool BWD>
static void hidden(const void* x, const void* dy, const void* w_in, const void* w_out, void* h, void* d, long long M, int C,
                   int F, hipStream_t stream) {
    const int nt = (int)up_div(F, 64);
    if constexpr (IO == KFH_BF16) {
        if (up_div(M, 128) * nt >= 256) {
            hipLaunchKernelGGL((ffn_hidden_kernel<IO, BWD, 128>), dim3(xcd_grid(up_div(M, 128), nt)), dim3(256), 0, stream, x,
                               dy, w_in, w_out, h, d, M, C, F);
            return;
        }
    }
    hipLaunchKernelGGL((ffn_hidden_kernel<IO, BWD, 64>), dim3(xcd_grid(up_div(M, 64), nt)), dim3(256), 0, stream, x, dy, w_in,
                       w_out, h, d, M, C, F);
}

template <int IO, int AK, int BK_, bool PART, int TM, int TN>
static void gemm(const void* A, long long lda, const void* B, long long ldb, void* out, long long Mo, int No, long long K,
                 long long kper, int splits, hipStream_t stream) {
    const long long mt = up_div(Mo, TM), nt = up_div(No, TN);
    hipLaunchKernelGGL((ffn_gemm_kernel<IO, AK, BK_, PART, TM, TN>),
                       dim3(PART ? xcd_grid(splits, (int)(mt * nt)) : xcd_grid(mt, (int)nt)), dim3(Waves<TM, TN>::NW * 64), 0,
                       stream, A, lda, B, ldb, out, Mo, No, K, kper, splits);
}

// out [Mo, No] = A [Mo, K] (AK) times B, [No, K] (K_MAJOR) or [K, No] (R_MAJOR); part: product_part_bytes
template <int IO, int AK, int BK_>
static void product(const void* A, long long lda, const void* B, long long ldb, void* out, float* part, long long Mo, int No,
                    long long K, hipStream_t stream) {
    const int splits = product_splits(Mo, No, K, IO);
    if (splits > 1) {
        const long long BK = IO == KFH_F32 ? 32 : 64, per = up_div(up_div(K, BK), splits) * BK;
        if constexpr (AK == K_MAJOR) gemm<IO, AK, BK_, true, 64, 64>(A, lda, B, ldb, part, Mo, No, K, per, splits, stream);
        sum_parts(part, splits, Mo * No, out, IO, stream);
        return;
    }
    const Tile t = pick_tile(Mo, No, 1, IO);
    if constexpr (IO == KFH_BF16) {
        if (t.n == 256) { gemm<IO, AK, BK_, false, 256, 256>(A, lda, B, ldb, out, Mo, No, K, K, 1, stream); return; }
        if (t.m == 256) { gemm<IO, AK, BK_, false, 256, 128>(A, lda, B, ldb, out, Mo, No, K, K, 1, stream); return; }
        if (t.m == 128) { gemm<IO, AK, BK_, false, 128, 128>(A, lda, B, ldb, out, Mo, No, K, K, 1, stream); return; }
    }
    if constexpr (AK == K_MAJOR) gemm<IO, AK, BK_, false, 64, 64>(A, lda, B, ldb, out, Mo, No, K, K, 1, stream);
}

// out [Ma, Nb] = A [M, Ma]^T B [M, Nb]; AK, BK_: R_MAJOR or R_BLOCK
template <int IO, int AK, int BK_>
static void wgrad(const void* A, int Ma, const void* B, int Nb, float* part, void* out, int out_dtype, long long M,
                  hipStream_t stream) {
    const Wgrad w = wgrad_plan(M, Ma, Nb, IO);
    auto run = [&](auto tm, auto tn) {
        gemm<IO, AK, BK_, true, decltype(tm)::v, decltype(tn)::v>(A, Ma, B, Nb, part, Ma, Nb, M, w.per, w.splits, stream);
    };
    bool done = false;
    if constexpr (IO == KFH_BF16) {
        done = true;
        if (w.t.m == 256 && w.t.n == 256) run(Int<256>{}, Int<256>{});
        else if (w.t.m == 256) run(Int<256>{}, Int<128>{});
        else if (w.t.n == 256) run(Int<128>{}, Int<256>{});
        else if (w.t.m == 128) run(Int<128>{}, Int<128>{});
        else done = false;
    }
    if (!done) run(Int<64>{}, Int<64>{});
    sum_parts(part, w.splits, (long long)Ma * Nb, out, out_dtype, stream);
}

// hidden values (and, up to C = 128, the second product) of a streamed call
template <int KS, bool BWD>
static void stream(const void* x, const void* dy, const void* w_in, const void* w_out, char* ws, const FfnWs& w, void* out,
                   long long M, int F, hipStream_t stream) {
    constexpr bool FUSE = KS <= 8;
    constexpr int NW = KS == 16 ? 8 : 4, OCC = BWD || KS == 16 ? 2 : 3;
    u32x4* pack = reinterpret_cast<u32x4*>(ws + w.pack);
    const long long slots = (long long)(F / 32) * stream_frags<KS, BWD, FUSE>() * 64;
    hipLaunchKernelGGL((ffn_pack_kernel<KS, BWD, FUSE>), dim3((unsigned)up_div(slots, 256)), dim3(256), 0, stream,
                       static_cast<const uint16_t*>(w_in), static_cast<const uint16_t*>(w_out), pack, F, slots);
    const long long tiles = up_div(M, 32 * NW);
    hipLaunchKernelGGL((ffn_stream_kernel<KS, BWD, FUSE, NW, OCC>), dim3((unsigned)tiles), dim3(NW * 64), 0, stream,
                       static_cast<const uint16_t*>(x), static_cast<const uint16_t*>(dy), pack,
                       reinterpret_cast<uint16_t*>(ws + w.h), reinterpret_cast<uint16_t*>(ws + w.d), static_cast<uint16_t*>(out), M, F);
}
template <bool BWD>
static void stream_by_width(int C, const void* x, const void* dy, const void* w_in, const void* w_out, char* ws,
                            const FfnWs& w, void* out, long long M, int F, hipStream_t s) {
    if (C == 64) stream<4, BWD>(x, dy, w_in, w_out, ws, w, out, M, F, s);
    else if (C == 128) stream<8, BWD>(x, dy, w_in, w_out, ws, w, out, M, F, s);
    else stream<16, BWD>(x, dy, w_in, w_out, ws, w, out, M, F, s);
}

template <int IO>
static void forward_t(const void* x, const void* w_in, const void* w_out, void* y, char* ws, long long M, int C, int F,
                      hipStream_t stream) {
    const FfnWs w = ffn_ws(M, C, F, 0, IO);
    const bool st = streamed(M, C, F, IO);
    if (st) stream_by_width<false>(C, x, nullptr, w_in, w_out, ws, w, y, M, F, stream);
    else hidden<IO, false>(x, nullptr, w_in, nullptr, ws + w.h, nullptr, M, C, F, stream);
    float* const part = reinterpret_cast<float*>(ws + w.part);
    if (!st) product<IO, K_MAJOR, K_MAJOR>(ws + w.h, F, w_out, F, y, part, M, C, F, stream);
    if constexpr (IO == KFH_BF16) {
        if (st && C > 128) product<IO, K_BLOCK, K_MAJOR>(ws + w.h, F, w_out, F, y, part, M, C, F, stream);
    }
}

template <int IO>
static void backward_t(const void* dy, const void* x, const void* w_in, const void* w_out, void* dx, void* dw_in,
                       void* dw_out, int dw_dtype, char* ws, long long M, int C, int F, hipStream_t stream) {
    const FfnWs w = ffn_ws(M, C, F, 1, IO);
    char* const h = ws + w.h;
    char* const d = ws + w.d;
    float* const part = reinterpret_cast<float*>(ws + w.part);
    const bool st = streamed(M, C, F, IO);
    if constexpr (IO == KFH_BF16) {
        if (st) {
            stream_by_width<true>(C, x, dy, w_in, w_out, ws, w, dx, M, F, stream);
            if (dw_out) wgrad<IO, R_MAJOR, R_BLOCK>(dy, C, h, F, part, dw_out, dw_dtype, M, stream);
            if (dw_in) wgrad<IO, R_BLOCK, R_MAJOR>(d, 2 * F, x, C, part, dw_in, dw_dtype, M, stream);
            if (dx && C > 128) product<IO, K_BLOCK, R_MAJOR>(d, 2LL * F, w_in, C, dx, part, M, C, 2LL * F, stream);
            return;
        }
    }
    hidden<IO, true>(x, dy, w_in, w_out, h, d, M, C, F, stream);
    if (dw_out) wgrad<IO, R_MAJOR, R_MAJOR>(dy, C, h, F, part, dw_out, dw_dtype, M, stream);
    if (dw_in) wgrad<IO, R_MAJOR, R_MAJOR>(d, 2 * F, x, C, part, dw_in, dw_dtype, M, stream);
    if (dx) product<IO, K_MAJOR, R_MAJOR>(d, 2LL * F, w_in, C, dx, part, M, C, 2LL * F, stream);
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
