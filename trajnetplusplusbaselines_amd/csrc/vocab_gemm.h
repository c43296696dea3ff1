// Matrix products of vocab_ce.hip: C[m, n] = sum_k A[m, k] B[n, k] on v_mfma_f32_32x32x16_f16, both operands fp16 in memory, either
// with k contiguous in a row ("KC") or with k as the row index ("KS": the transposing LDS read hands the matrix core its layout, so
// no transposed copy of anything is ever made).
//
// SPLIT operands carry fp32 values as two fp16 numbers, x = hi + lo (22 bits; what is left is below 2^-22 of x), stored as blocks of
// 32 values: 32 hi | 32 lo.  A product is hi*hi + hi*lo + lo*hi, three matrix instructions into one fp32 accumulator: 2500 / 3
// TFLOP/s of matrix rate where v_mfma_f32_* has 157.
//
// A step stages 128 bytes per tile row (64 values, or 32 split ones) by global_load_lds into one of two LDS buffers while the other
// is multiplied.  global_load_lds writes linearly, so the bank swizzle is applied to the global address: KC rows of 128 bytes put
// chunk c (16 bytes) at c ^ ((row >> 1) & 7): sixteen consecutive rows cover all 64 banks; KS rows put 64-byte unit u at
// u ^ (row & 3): the four k rows of a transposing read cover all 64 banks.
#pragma once
#include "vocab_types.h"

#include <type_traits>

namespace tnp {

typedef half_t half8 __attribute__((ext_vector_type(8)));
typedef short short4v __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

#define TNP_LDS __attribute__((address_space(3)))
#define TNP_GLB __attribute__((address_space(1)))

struct GemmOperand {
    const half_t *p;     // first element of the matrix
    int64_t ld;          // stored elements per row (a multiple of 64)
    int64_t rows;        // rows that may be read: a row index beyond is clamped to the last
    int perm;            // KS: bits 2 and 3 of the row index change places (the order in which the G kernel stores its columns)
};

// One operand's tile of BR rows (KC) / BR columns (KS).
template <bool KS, bool SPLIT, int BR, int NW> struct TileStage {
    static constexpr int INSTR = BR / 8 / NW;                      // 1 KB wave instructions per wave and step
    static_assert(BR / 8 % NW == 0, "tile rows must spread evenly over the waves");
    static constexpr int KSTEP = SPLIT ? 32 : 64;
    const half_t *base;
    int64_t ld, rows, row0;
    uint32_t off[INSTR];
    int perm;

    // KC: tile rows [r0, r0 + BR), k from stored column c0.  KS: tile columns (stored) from c0, k from row r0.
    __device__ __forceinline__ void init(const GemmOperand &o, int64_t r0, int64_t c0, int wave, int lane) {
        ld = o.ld; rows = o.rows; perm = o.perm; row0 = r0;
        if (!KS) {
            base = o.p + r0 * ld + c0;
#pragma unroll
            for (int j = 0; j < INSTR; ++j) {
                const int r = (wave + j * NW) * 8 + (lane >> 3);
                const int64_t row = r0 + r < rows ? r : rows - 1 - r0;
                off[j] = (uint32_t)(row * ld) + ((lane & 7) ^ ((r >> 1) & 7)) * 8;
            }
        } else {
            base = o.p;
            constexpr int CB = BR * 2 * (SPLIT ? 2 : 1);           // bytes per k row
#pragma unroll
            for (int j = 0; j < INSTR; ++j) {
                const int byte = (wave + j * NW) * 1024 + lane * 16, r = byte / CB, ch = byte % CB / 16;
                const int64_t col = c0 + (ch ^ ((r & 3) << 2)) * 8;
                off[j] = (uint32_t)(col < ld - 8 ? col : ld - 8);
            }
        }
    }
    __device__ __forceinline__ void load(int step, char *lds, int wave, int lane) const {
#pragma unroll
        for (int j = 0; j < INSTR; ++j) {
            const half_t *src;
            if (!KS) {
                src = base + (int64_t)step * 64 + off[j];
            } else {
                constexpr int CB = BR * 2 * (SPLIT ? 2 : 1);
                int r = ((wave + j * NW) * 1024 + lane * 16) / CB;
                if (perm) r = (r & ~12) | ((r & 4) << 1) | ((r & 8) >> 1);
                int64_t row = row0 + (int64_t)step * KSTEP + r;
                row = row < rows ? row : rows - 1;
                src = base + row * ld + off[j];
            }
            __builtin_amdgcn_global_load_lds((const TNP_GLB void *)src, (TNP_LDS void *)(lds + (wave + j * NW) * 1024), 16, 0, 0);
        }
    }
    // operand of one 32-row block at tile row r0, sub-step ss of 16 values, plane 0 = hi / 1 = lo (SPLIT)
    static __device__ __forceinline__ half8 frag(const char *lds, int r0, int ss, int plane, int lane) {
        if (!KS) {
            const int r = r0 + (lane & 31), ch = (SPLIT ? plane * 4 : 0) + ss * 2 + (lane >> 5);
            return *(const half8 *)(lds + r * 128 + ((ch ^ ((r >> 1) & 7)) * 16));
        } else {
            return half8{};                                        // KS operands come through ks_frags
        }
    }
    static constexpr int CB = BR * 2 * (SPLIT ? 2 : 1);            // bytes per k row of a KS tile
    // KS: LDS byte address of the first value this lane fetches for 32 columns from c (stored), k rows 0 .. 3 of its half.  Rows
    // row, row + 4, row + 16 share (row & 3), hence the swizzle: further rows are constant offsets.
    static __device__ __forceinline__ uint32_t ks_addr(const char *lds, int c, int lane) {
        const int g = lane >> 4, j = lane & 15, row = 8 * (g >> 1) + (j >> 2), col = c + 16 * (g & 1) + 4 * (j & 3);
        return (uint32_t)(uintptr_t)(TNP_LDS const char *)lds + row * CB + (((col >> 3) ^ ((row & 3) << 2)) * 16) + (col & 7) * 2;
    }
};

// Two 32-column blocks of a KS tile, k values 16 ss .. 16 ss + 15 (OFF = 16 ss rows in bytes).  One asm block that ends with its own
// wait: as builtins these reads would first wait for every global_load_lds in flight, that is for the NEXT step's tile.
template <int OFF, int CB>
__device__ __forceinline__ void ks_read2(uint32_t a0, uint32_t a1, half8 &f0, half8 &f1) {
    typedef int int2v __attribute__((ext_vector_type(2)));
    typedef int int4v __attribute__((ext_vector_type(4)));
    int2v p0, q0, p1, q1;
    asm volatile("ds_read_b64_tr_b16 %0, %4 offset:%c6\n\t"
                 "ds_read_b64_tr_b16 %1, %4 offset:%c7\n\t"
                 "ds_read_b64_tr_b16 %2, %5 offset:%c6\n\t"
                 "ds_read_b64_tr_b16 %3, %5 offset:%c7\n\t"
                 "s_waitcnt lgkmcnt(0)"
                 : "=&v"(p0), "=&v"(q0), "=&v"(p1), "=&v"(q1)
                 : "v"(a0), "v"(a1), "i"(OFF), "i"(OFF + 4 * CB)
                 : "memory");
    f0 = __builtin_bit_cast(half8, int4v{p0.x, p0.y, q0.x, q0.y});
    f1 = __builtin_bit_cast(half8, int4v{p1.x, p1.y, q1.x, q1.y});
}
template <int OFF, int CB>
__device__ __forceinline__ void ks_read4(uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, half8 &f0, half8 &f1, half8 &f2, half8 &f3) {
    typedef int int2v __attribute__((ext_vector_type(2)));
    typedef int int4v __attribute__((ext_vector_type(4)));
    int2v p0, q0, p1, q1, p2, q2, p3, q3;
    asm volatile("ds_read_b64_tr_b16 %0, %8 offset:%c12\n\t"
                 "ds_read_b64_tr_b16 %1, %8 offset:%c13\n\t"
                 "ds_read_b64_tr_b16 %2, %9 offset:%c12\n\t"
                 "ds_read_b64_tr_b16 %3, %9 offset:%c13\n\t"
                 "ds_read_b64_tr_b16 %4, %10 offset:%c12\n\t"
                 "ds_read_b64_tr_b16 %5, %10 offset:%c13\n\t"
                 "ds_read_b64_tr_b16 %6, %11 offset:%c12\n\t"
                 "ds_read_b64_tr_b16 %7, %11 offset:%c13\n\t"
                 "s_waitcnt lgkmcnt(0)"
                 : "=&v"(p0), "=&v"(q0), "=&v"(p1), "=&v"(q1), "=&v"(p2), "=&v"(q2), "=&v"(p3), "=&v"(q3)
                 : "v"(a0), "v"(a1), "v"(a2), "v"(a3), "i"(OFF), "i"(OFF + 4 * CB)
                 : "memory");
    f0 = __builtin_bit_cast(half8, int4v{p0.x, p0.y, q0.x, q0.y});
    f1 = __builtin_bit_cast(half8, int4v{p1.x, p1.y, q1.x, q1.y});
    f2 = __builtin_bit_cast(half8, int4v{p2.x, p2.y, q2.x, q2.y});
    f3 = __builtin_bit_cast(half8, int4v{p3.x, p3.y, q3.x, q3.y});
}
// N = 2 or 4 blocks at the addresses a[0 .. N)
template <int OFF, int CB, int N> __device__ __forceinline__ void ks_frags(const uint32_t (&a)[N], half8 (&f)[N]) {
    static_assert(N == 2 || N == 4, "two or four blocks of 32 columns per wave");
    if constexpr (N == 2) ks_read2<OFF, CB>(a[0], a[1], f[0], f[1]);
    else ks_read4<OFF, CB>(a[0], a[1], a[2], a[3], f[0], f[1], f[2], f[3]);
}

// Accumulates steps [s0, s1) of tile (a at row / column a0, b at b0) into acc.  KC operands start at stored column ak0 / bk0, KS
// operands at row ak0 / bk0.  LDS: 2 * (BM + BN) * 128 bytes.
template <bool SPLIT, bool A_KS, bool B_KS, int BM, int BN, int WM, int WN>
__device__ __forceinline__ void gemm_tile(const GemmOperand &a, const GemmOperand &b, int64_t a0, int64_t ak0, int64_t b0, int64_t bk0, int s0,
                                          int s1, char *lds, f32x16 (&acc)[BM / WM / 32][BN / WN / 32]) {
    constexpr int NW = WM * WN, TM = BM / WM / 32, TN = BN / WN / 32, STAGE = (BM + BN) * 128;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WN, wn = wave % WN;
    typedef TileStage<A_KS, SPLIT, BM, NW> SA;
    typedef TileStage<B_KS, SPLIT, BN, NW> SB;
    SA sa;
    SB sb;
    if (A_KS) sa.init(a, ak0, a0 * (SPLIT ? 2 : 1), wave, lane); else sa.init(a, a0, ak0, wave, lane);
    if (B_KS) sb.init(b, bk0, b0 * (SPLIT ? 2 : 1), wave, lane); else sb.init(b, b0, bk0, wave, lane);
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.0f;
    if (s0 >= s1) return;
    sa.load(s0, lds, wave, lane);
    sb.load(s0, lds + BM * 128, wave, lane);
    __syncthreads();
    for (int s = s0; s < s1; ++s) {
        char *cur = lds + ((s - s0) & 1) * STAGE, *nxt = lds + ((s - s0 + 1) & 1) * STAGE;
        if (s + 1 < s1) {
            sa.load(s + 1, nxt, wave, lane);
            sb.load(s + 1, nxt + BM * 128, wave, lane);
        }
        const char *la = cur, *lb = cur + BM * 128;
        constexpr int P = SPLIT ? 2 : 1, SS = SPLIT ? 2 : 4;
        uint32_t aa[P][TM], ab[P][TN];                             // KS operands: LDS addresses
        if (A_KS)
#pragma unroll
            for (int p = 0; p < P; ++p)
#pragma unroll
                for (int i = 0; i < TM; ++i) aa[p][i] = SA::ks_addr(la, (wm * TM + i) * 32 * P + p * 32, lane);
        if (B_KS)
#pragma unroll
            for (int p = 0; p < P; ++p)
#pragma unroll
                for (int j = 0; j < TN; ++j) ab[p][j] = SB::ks_addr(lb, (wn * TN + j) * 32 * P + p * 32, lane);
        auto sub = [&](auto ssc) {
            constexpr int ss = decltype(ssc)::value;
            half8 fa[P][TM], fb[P][TN];
#pragma unroll
            for (int p = 0; p < P; ++p) {
                if constexpr (A_KS) ks_frags<ss * 16 * SA::CB, SA::CB, TM>(aa[p], fa[p]);
                else
#pragma unroll
                    for (int i = 0; i < TM; ++i) fa[p][i] = SA::frag(la, (wm * TM + i) * 32, ss, p, lane);
                if constexpr (B_KS) ks_frags<ss * 16 * SB::CB, SB::CB, TN>(ab[p], fb[p]);
                else
#pragma unroll
                    for (int j = 0; j < TN; ++j) fb[p][j] = SB::frag(lb, (wn * TN + j) * 32, ss, p, lane);
            }
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int j = 0; j < TN; ++j) {
                    if constexpr (SPLIT) {                         // the small products first: they are not lost against the large ones
                        acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fa[1][i], fb[0][j], acc[i][j], 0, 0, 0);
                        acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fa[0][i], fb[1][j], acc[i][j], 0, 0, 0);
                    }
                    acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fa[0][i], fb[0][j], acc[i][j], 0, 0, 0);
                }
        };
        sub(std::integral_constant<int, 0>());
        sub(std::integral_constant<int, 1>());
        if constexpr (SS == 4) {
            sub(std::integral_constant<int, 2>());
            sub(std::integral_constant<int, 3>());
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");            // the next step's tile has landed
        __syncthreads();
    }
}

// Workgroup -> tile: the eight XCDs take the workgroups in turn, so each gets a contiguous share of the tiles, walked in groups of
// eight tile rows; the panels of a group stay in the XCD's own L2.  Returns false for the workgroups behind the last tile.
__device__ __forceinline__ bool gemm_tile_of(int bid, int tiles_m, int tiles_n, int &tm, int &tn) {
    const int total = tiles_m * tiles_n, per = (total + 7) / 8;
    const int t = (bid & 7) * per + (bid >> 3);
    if ((bid >> 3) >= per || t >= total) return false;
    const int width = 8 * tiles_n, g = t / width, first = g * 8;
    const int h = tiles_m - first < 8 ? tiles_m - first : 8, r = t - g * width;
    tm = first + r % h;
    tn = r / h;
    return true;
}
inline int gemm_grid(int64_t tiles) { return (int)((tiles + 7) / 8 * 8); }

}  // namespace tnp
