// Operand and result tiles of the gated feed-forward block's matrix products (gatedffn.hip,
// gatedffn_stream.hip).
#pragma once
#include "train.hpp"

namespace kfh {

template <int V> struct Int { static constexpr int v = V; };

// ---------------------------------------------------------------------------------------------
// Operand tiles.  A tile of ROWS x BK bf16 operand values (rows: output index, k: contraction), in P
// parts (planes `plane` bytes apart; P = 3: split3 parts of fp32 values), goes from memory to registers
// (fetch) to LDS (commit), where it is stored [part][row][BK + 8], so that the 8 k-consecutive values of
// an MFMA fragment are one 16-byte read; the 8 values of padding keep consecutive rows on different banks.
//   K_MAJOR : memory is [row][k], k contiguous: a unit is 8 k of a row
//   R_MAJOR : memory is [k][row], rows contiguous: a unit is 4 k x 8 rows, written transposed, 4 k
//             (8 bytes) per row
//   K_BLOCK, R_BLOCK: the same two for hidden values written by ffn_stream_kernel, blocks of 32 rows x
//             32 channels (ld: channels) of two MFMA fragments each: hidden_slot
// Values outside [row < rmax, k < kmax] are zeros: their addresses are kept inside the tensor, so that
// no load sits behind a branch, and the values cleared when they are committed.
// ---------------------------------------------------------------------------------------------
enum : int { K_MAJOR = 0, R_MAJOR, K_BLOCK, R_BLOCK };

// 16-byte slot of the 8 channels 16 ks + 4 half + {0..3, 8..11} of block (m / 32, channel block hb), row m
__device__ __forceinline__ size_t hidden_slot(long long m, int hb, int nhb, int ks, int half) {
    return ((size_t)((m >> 5) * nhb + hb) * 2 + ks) * 64 + half * 32 + (m & 31);
}

template <int KIND, int ROWS, int BK, int P, int NT>
struct TileLoad {
    static constexpr bool KC = KIND == K_MAJOR || KIND == K_BLOCK;
    static constexpr int LDK = BK + 8;                       // bf16 per stored row
    static constexpr int UNITS1 = KC ? ROWS * BK / 8 : ROWS * BK / 32;      // of a part
    static constexpr int UNITS = P * UNITS1;
    static constexpr int NU = (UNITS + NT - 1) / NT;         // units per thread
    static constexpr int NV = KC ? 1 : 4;                    // 16-byte vectors per unit
    struct Regs {                                            // a tile on its way from memory to LDS
        u32x4 v[NU][NV];
        unsigned bad;                                        // bit i * NV + j: vector j of unit i lies outside
    };
    const char* base;                                        // of the tile's first row; the same in all lanes
    long long step, vec;                                     // bytes from a k to the next, from a vector of a unit to the next
    uint32_t off[NU];                                        // bytes from base of unit i at k = 0
    long long part[P > 1 ? NU : 1];                          // bytes from the first part's plane
    unsigned off_rows;                                       // as Regs::bad, for rows behind the last

    static __device__ __forceinline__ int unit(int i, int tid) {
        const int u = i * NT + tid;
        return UNITS % NT ? min(u, UNITS - 1) : u;
    }
    // k of unit u (of a part) inside the tile
    static __device__ __forceinline__ int unit_k(int u) {
        return KIND == K_MAJOR ? (u % (BK / 8)) * 8 : KIND == K_BLOCK ? (u / ROWS) * 8 : (u % (BK / 4)) * 4;
    }
    // what does not change along the contraction: every later address is base + k * step + off + j * vec.
    // A row behind the last reads the last one's values, which commit clears.
    __device__ __forceinline__ void init(const void* src, long long ld, long long plane, long long row0, long long rmax,
                                         int tid) {
        const int left = (int)min(rmax - row0, (long long)ROWS);          // rows of this tile
        const int nhb = (int)(ld >> 5);
        off_rows = 0;
        const char* const s = static_cast<const char*>(src);
        if constexpr (KIND == K_MAJOR) { base = s + row0 * ld * 2; step = 2; vec = 0; }
        else if constexpr (KIND == R_MAJOR) { base = s + row0 * 2; step = vec = ld * 2; }
        else if constexpr (KIND == K_BLOCK) { base = s + (row0 >> 5) * nhb * 2048; step = 64; vec = 0; }   // 32 k: 2 KiB
        else { base = s + (row0 >> 5) * 2048; step = (long long)nhb * 64; vec = 16; }                       // 32 k: nhb blocks
#pragma unroll
        for (int i = 0; i < NU; ++i) {
            const int ua = unit(i, tid), u = P > 1 ? ua % UNITS1 : ua, k = unit_k(u);
            if constexpr (P > 1) part[i] = (ua / UNITS1) * plane;
            int r = KIND == K_MAJOR ? u / (BK / 8) : KIND == K_BLOCK ? u % ROWS : (u / (BK / 4)) * 8;
            if (r >= left) {
                off_rows |= ((1u << NV) - 1) << (i * NV);
                r = KC ? left - 1 : left - 8;
            }
            if constexpr (KIND == K_MAJOR) off[i] = (uint32_t)(r * (int)ld + k) * 2;
            else if constexpr (KIND == R_MAJOR) off[i] = (uint32_t)(k * (int)ld + r) * 2;
            else if constexpr (KIND == K_BLOCK)
                off[i] = (uint32_t)(((r >> 5) * nhb + (k >> 5)) * 128 + ((k >> 3) & 3) * 32 + (r & 31)) * 16;
            else
                off[i] = (uint32_t)(((k >> 5) * nhb + (r >> 5)) * 128 + ((r >> 3) & 3) * 32 + (k & 31)) * 16;
        }
    }
    __device__ __forceinline__ u32x4 get(const char* b, uint32_t o, int i) const {
        if constexpr (P > 1) b += part[i];
        return *reinterpret_cast<const u32x4*>(b + o);
    }
    // the tile at k0 < kmax; only a tile that reaches behind kmax looks at single vectors (they read the
    // tile's first k instead, which lies inside)
    __device__ __forceinline__ void fetch(long long k0, long long kmax, int tid, Regs& t) const {
        const char* const b = base + k0 * step;
        t.bad = off_rows;
        if (k0 + BK <= kmax) {
#pragma unroll
            for (int i = 0; i < NU; ++i)
#pragma unroll
                for (int j = 0; j < NV; ++j) t.v[i][j] = get(b + j * vec, off[i], i);
        } else {
#pragma unroll
            for (int i = 0; i < NU; ++i) {
                const int ua = unit(i, tid), k = unit_k(P > 1 ? ua % UNITS1 : ua);
                // off of the same row at k = 0
                uint32_t first = off[i];
                if constexpr (KIND == K_MAJOR || KIND == R_MAJOR) first -= (uint32_t)(k * step);
                else if constexpr (KIND == K_BLOCK) first -= (uint32_t)((k >> 5) * 128 + ((k >> 3) & 3) * 32) * 16;
                else first -= (uint32_t)((k >> 5) * 32 * step) + (k & 31) * 16;
#pragma unroll
                for (int j = 0; j < NV; ++j) {
                    const bool out = k0 + k + j >= kmax;
                    t.bad |= (unsigned)out << (i * NV + j);
                    t.v[i][j] = get(out ? b : b + j * vec, out ? first : off[i], i);
                }
            }
        }
    }
    static __device__ __forceinline__ void commit(uint16_t* lds, int tid, Regs& t) {
        if (t.bad) {
#pragma unroll
            for (int i = 0; i < NU; ++i)
#pragma unroll
                for (int j = 0; j < NV; ++j)
                    if ((t.bad >> (i * NV + j)) & 1) t.v[i][j] = u32x4{0u, 0u, 0u, 0u};
        }
#pragma unroll
        for (int i = 0; i < NU; ++i) {
            const int ua = i * NT + tid;
            if (UNITS % NT != 0 && ua >= UNITS) continue;
            const int u = P > 1 ? ua % UNITS1 : ua;
            uint16_t* const l = lds + (P > 1 ? (ua / UNITS1) * ROWS * LDK : 0);
            const u32x4(&v)[NV] = t.v[i];
            if constexpr (KIND == K_MAJOR) {
                *reinterpret_cast<u32x4*>(l + (u / (BK / 8)) * LDK + (u % (BK / 8)) * 8) = v[0];
            } else if constexpr (KIND == K_BLOCK) {
                const int g = u / ROWS;                      // group 4 b + 2 ks + half: channels 32 b + 16 ks + 4 half + {0..3, 8..11}
                uint16_t* d = l + (u % ROWS) * LDK + (g >> 1) * 16 + (g & 1) * 4;
                *reinterpret_cast<u32x2*>(d) = u32x2{v[0][0], v[0][1]};
                *reinterpret_cast<u32x2*>(d + 8) = u32x2{v[0][2], v[0][3]};
            } else {
                const int g = u / (BK / 4);
                uint16_t* const d = l + (KIND == R_BLOCK ? (g >> 1) * 16 + (g & 1) * 4 : g * 8) * LDK + (u % (BK / 4)) * 4;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    // half-word e of the four vectors
                    const uint32_t a = v[0][e >> 1], b = v[1][e >> 1], c = v[2][e >> 1], f = v[3][e >> 1];
                    const u32x2 w = (e & 1) ? u32x2{(a >> 16) | (b & 0xffff0000u), (c >> 16) | (f & 0xffff0000u)}
                                            : u32x2{(a & 0xffffu) | (b << 16), (c & 0xffffu) | (f << 16)};
                    *reinterpret_cast<u32x2*>(d + (KIND == R_BLOCK ? 8 * (e >> 2) + (e & 3) : e) * LDK) = w;
                }
            }
        }
    }
};

// acc[i][j] += rows (a0 + 32 i) of tile `ta` times rows (b0 + 32 j) of tile `tb` over BK, as
// D[row of b][column = row of a]: a lane then holds four consecutive b indices of one a row.
template <int P, int NA, int NB, int AROWS, int BROWS, int BK>
__device__ __forceinline__ void tile_mma(const uint16_t* ta, int a0, const uint16_t* tb, int b0, int lane,
                                         f32x16 (&acc)[NA][NB]) {
    constexpr int LDK = BK + 8;
    const int col = lane & 31, half = lane >> 5;
#pragma unroll
    for (int ks = 0; ks < BK / 16; ++ks) {
        bf16x8 a[NA][P], b[NB][P];
#pragma unroll
        for (int p = 0; p < P; ++p) {
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
                if constexpr (P == 1) {
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
// row tile follow each other on one XCD, so its rows are read from memory once.  With few row tiles, unless they
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
template <int IO, int RM, int RN, int NT>
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

// ---- rows in registers (gatedffn_stream.hip) ------------------------------------------------
size_t ffn_stream_pack_bytes(int C, int F, int backward);
// dy null: forward, out = y (C <= 128) or h in blocks (C = 256); else d and h in blocks, out = dx (C <= 128, may be null)
void launch_ffn_stream(const void* x, const void* dy, const void* w_in, const void* w_out, void* pack, void* h, void* d,
                       void* out, long long M, int C, int F, hipStream_t stream);

}  // namespace kfh
